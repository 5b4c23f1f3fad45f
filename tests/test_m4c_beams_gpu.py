"""M4C's beam search over the paged cache (`num_beams`, mmf_amd/models/m4c.py `_decode_beams`) against a search made with the CPU oracle, which re-runs the whole model for
every hypothesis and step (teacher forcing, as the reference's greedy loop does, mmf/models/m4c.py:284-304)."""
import functools

import pytest
import torch

from mmf_amd.common.sample import SampleList
from oracle import m4c_oracle as O
from tests.golden_utils import load_m4c_case
from tests.model_utils import build_m4c, sample_to

BOS, EOS = 1, 2


def repeat(sample, W):
    return {k: (v.repeat_interleave(W, 0) if torch.is_tensor(v) else {n: x.repeat_interleave(W, 0) for n, x in v.items()} if isinstance(v, dict) else v) for k, v in sample.items()}


def oracle_scores(sd, cfg, sample, tokens):
    """Scores [B, W, D, V + N] of hypotheses `tokens` [B, W, D] (column t feeds step t + 1)."""
    B, W, D = tokens.shape
    s = repeat(sample, W)
    prev = torch.zeros(B * W, D, dtype=torch.long)
    prev[:, 0] = BOS
    prev[:, 1:] = tokens.view(B * W, D)[:, :-1]
    s["train_prev_inds"] = prev
    with torch.no_grad():
        return O.m4c_forward(sd, cfg, s, training_mode=True)["scores"].view(B, W, D, -1)


@functools.lru_cache(None)
def oracle_search(W):
    z, case, cfg, sd, sample = load_m4c_case()
    B, D = sample["train_prev_inds"].shape
    tokens = torch.zeros(B, W, D, dtype=torch.long)
    score = torch.full((B, W), float("-inf"), dtype=torch.float64)
    score[:, 0] = 0
    done = torch.zeros(B, W, dtype=torch.bool)
    gap = float("inf")
    for t in range(D):
        x = torch.log_softmax(oracle_scores(sd, cfg, sample, tokens)[:, :, t].double(), -1)
        V = x.shape[-1]
        cand = score[:, :, None] + x
        only = torch.full_like(cand, float("-inf"))
        only[:, :, EOS] = score
        cand = torch.where(done[:, :, None], only, cand).view(B, -1)
        v, i = torch.sort(cand, dim=1, descending=True, stable=True)
        gap = min(gap, float((v[:, :W] - v[:, 1:W + 1]).min()))
        score, parent, tok = v[:, :W], i[:, :W] // V, i[:, :W] % V
        tokens = tokens.gather(1, parent[:, :, None].expand_as(tokens)).clone()
        tokens[:, :, t] = tok
        done = done.gather(1, parent) | (tok == EOS)
    return tokens, score, gap


@pytest.mark.parametrize("W", [1, 3, 5])
def test_the_oracle_search_decides_its_order(W):
    assert oracle_search(W)[2] > 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("W", [1, 3, 5])
def test_beam_search_finds_what_the_oracle_finds(W):
    import mmf_amd
    z, case, cfg, sd, sample = load_m4c_case()
    want, score, _ = oracle_search(W)
    model = build_m4c(cfg, sd, num_beams=W).eval()
    with torch.no_grad(), mmf_amd.fp32_inference():
        out = model(SampleList(sample_to(sample, "cuda")))
    assert torch.equal(out["beam_tokens"].cpu(), want)
    assert float((out["beam_scores"].cpu().double() - score).abs().max()) < 1e-3            # the fp32 path's bound on scores (1e-3), over the few steps
    ref = oracle_scores(sd, cfg, sample, want[:, :1])[:, 0]
    got = out["scores"].cpu()
    valid = ref > -5000
    assert got.shape == ref.shape and float((got - ref).abs()[valid].max()) < 1e-3 and bool((got[~valid] < -5000).all())


@pytest.mark.gpu
def test_beam_search_in_bf16_scores_its_hypotheses_like_the_oracle_and_greedy_is_unchanged():
    z, case, cfg, sd, sample = load_m4c_case()
    tol = 5e-2                                       # the bf16 bound of every M4C parity test
    model = build_m4c(cfg, sd, num_beams=4).eval()
    with torch.no_grad():
        out = model(SampleList(sample_to(sample, "cuda")))
    tokens = out["beam_tokens"].cpu()
    ref = oracle_scores(sd, cfg, sample, tokens)
    got, best = out["scores"].float().cpu(), ref[:, 0]
    valid = best > -5000
    assert float((got - best).abs()[valid].max()) <= tol * (1 + float(best[valid].abs().max()))
    # the score of every hypothesis, from the oracle's scores along its tokens: steps behind an end token add nothing
    logp = torch.log_softmax(ref.double(), -1).gather(3, tokens[..., None])[..., 0]
    after = torch.cat([torch.zeros_like(tokens[:, :, :1]), (tokens == EOS).long().cumsum(2)[:, :, :-1]], 2) > 0
    total = logp.masked_fill(after, 0).sum(2)
    D = tokens.shape[2]
    assert float((out["beam_scores"].cpu().double() - total).abs().max()) <= 2 * D * tol * (1 + float(best[valid].abs().max()))
    assert bool((out["beam_scores"][:, :-1] >= out["beam_scores"][:, 1:]).all())
    model.config["num_beams"] = 0
    with torch.no_grad():
        a = model(SampleList(sample_to(sample, "cuda")))
    with torch.no_grad():
        b = build_m4c(cfg, sd).eval()(SampleList(sample_to(sample, "cuda")))
    assert set(a) == set(b) and torch.equal(a["scores"], b["scores"])


@pytest.mark.gpu
def test_one_beam_at_the_textvqa_shape_is_the_greedy_loop():
    """20 + 100 + 50 encoder positions, 12 steps, 5000 + 50 scores: until a sample's first end token or undecided step, one beam takes the greedy choices."""
    import warnings

    from mmf_amd.common.registry import registry
    from mmf_amd.utils.configuration import Config
    registry.register("config", Config({"datasets": "textvqa"}))
    registry.register("textvqa_num_final_outputs", 5050)
    registry.register("textvqa_answer_processor", Config({"BOS_IDX": 1}))
    torch.manual_seed(23)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        model = registry.get_model_class("m4c")(Config({"model": "m4c", "text_bert_init_from_bert_base": False}))
        model.build(); model.init_losses()
    model = model.to("cuda").eval()
    with torch.no_grad():       # well separated choices (random init gives near-ties)
        model.classifier.module.weight.mul_(8.0); model.ocr_ptr_net.query.weight.mul_(8.0); model.ocr_ptr_net.key.weight.mul_(8.0)
    B, D = 6, 12
    g = torch.Generator().manual_seed(6)
    sample = {
        "text": torch.randint(1, 30522, (B, 20), generator=g), "text_len": torch.randint(3, 21, (B,), generator=g),
        "image_feature_0": torch.rand(B, 100, 2048, generator=g), "obj_bbox_coordinates": torch.rand(B, 100, 4, generator=g),
        "image_info_0": {"max_features": torch.randint(10, 101, (B,), generator=g)},
        "context_feature_0": torch.randn(B, 50, 300, generator=g), "context_feature_1": torch.rand(B, 50, 604, generator=g),
        "image_feature_1": torch.rand(B, 100, 2048, generator=g), "ocr_bbox_coordinates": torch.rand(B, 50, 4, generator=g),
        "context_info_0": {"max_features": torch.randint(1, 51, (B,), generator=g)}, "order_vectors": torch.zeros(B, 50, 50),
        "train_prev_inds": torch.zeros(B, D, dtype=torch.long), "targets": torch.zeros(B, D, 5050),
        "train_loss_mask": torch.ones(B, D), "dataset_name": "textvqa", "dataset_type": "val"}
    batch = SampleList(sample_to(sample, "cuda"))
    with torch.no_grad():
        greedy = model(batch)["scores"].float()
        model.config["num_beams"] = 1
        one = model(batch)
        model.config["num_beams"] = 5
        five = model(batch)
    top2 = greedy.topk(2, dim=-1)
    decided = (top2.values[..., 0] - top2.values[..., 1]) > 0.5              # steps whose choice is not a bf16-noise tie
    assert bool(decided.float().mean() > 0.5)
    for b in range(B):
        n = 0
        while n < D and bool(decided[b, n]) and int(top2.indices[b, n, 0]) != EOS:
            n += 1
        assert torch.equal(one["beam_tokens"][b, 0, :n], top2.indices[b, :n, 0]), b
    assert tuple(five["beam_tokens"].shape) == (B, 5, D) and tuple(five["scores"].shape) == (B, D, 5050)
    assert bool(torch.isfinite(five["beam_scores"]).all())
