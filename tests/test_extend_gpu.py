"""Going on with cached sequences: Qwen2Decoder.extend, forward() with several new tokens behind a populated cache, prompts in portions beside decode steps
(ContinuousBatcher(prefill_chunk=...)) and stretched rotary frequencies, against the oracle's whole prompts."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import omchat_oracle as O  # noqa: E402
from tiny import TINY, tiny_inputs, tiny_state_dict  # noqa: E402
from test_model_gpu import check, oracle_cfg, tiny_cfgs  # noqa: E402
from test_serving_gpu import _same_or_near_tie  # noqa: E402


@pytest.fixture(scope="module")
def sd():
    return {k: v.to(torch.bfloat16).float() for k, v in tiny_state_dict(0).items()}


def _model(sd, **kw):
    from omchat_b200.model.omchat import OmChatQwen2ForCausalLM
    return OmChatQwen2ForCausalLM.from_state_dict(sd, tiny_cfgs(**kw), device="cuda")


@pytest.fixture(scope="module")
def model(sd):
    return _model(sd)


def _ids(n, seed):
    return torch.randint(1, TINY["vocab"], (1, n), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("stream", [True, False])
@pytest.mark.parametrize("portions", [(1, 5, 30, 1, 63, 20), (70, 50), (3, 117)])
def test_portions_of_a_prompt_are_the_prompt(model, sd, portions, stream):
    """Every position's logits, portion by portion (few rows: the streaming GEMMs, or the ones of a prompt), and a decode step behind them."""
    dec, n = model.model.decoder, sum(portions)
    ids = _ids(n + 1, 3)
    want, _, _, _ = O.forward_multimodal(ids, None, sd, oracle_cfg())
    cache = dec.new_cache(1, 200)
    embeds = dec.w.embed[ids[0, :n].cuda()]
    was, dec.stream_enabled = dec.stream_enabled, stream
    try:
        first = 0
        for m in portions:
            rows = embeds[first:first + m].clone()
            got = dec.extend(rows, [0, m], cache, logits="all")
            assert torch.equal(rows, embeds[first:first + m])           # the caller's rows are not the residual stream
            check(got, want[0, first:first + m], f"portion of {m} at {first}")
            first += m
            assert cache.host_lens == [first] and cache.ctx_lens.tolist() == [first]
    finally:
        dec.stream_enabled = was
    check(dec.decode_step(ids[0, n:].cuda(), cache), want[0, n:], "decode step behind the portions")


def test_sequences_of_many_lengths(model, sd):
    """Chunks of none, one and many tokens behind contexts of many lengths, for some rows of a cache; the others keep their state."""
    dec = model.model.decoder
    cache = dec.new_cache(4, 128)
    have, new = [17, 0, 40, 64], [3, 33, 0, 1]
    ids = [_ids(h + n + 1, 10 + i) for i, (h, n) in enumerate(zip(have, new))]
    rows = lambda parts: torch.cat([dec.w.embed[p.cuda()] for p in parts])  # noqa: E731
    offs = lambda lens: [0] + torch.tensor(lens).cumsum(0).tolist()  # noqa: E731
    dec.extend(rows([x[0, :h] for x, h in zip(ids, have)]), offs(have), cache, logits="none")
    order = [3, 0, 1]
    got = dec.extend(rows([ids[s][0, have[s]:have[s] + new[s]] for s in order]), offs([new[s] for s in order]), cache, logits="last", slots=order)
    for i, s in enumerate(order):
        want = O.forward_multimodal(ids[s][:, :have[s] + new[s]], None, sd, oracle_cfg())[0]
        check(got[i:i + 1], want[0, -1:], f"cache row {s}")
    assert cache.host_lens == [20, 33, 40, 65] and cache.ctx_lens.tolist() == [20, 33, 40, 65]
    assert dec.extend(rows([ids[2][0, :0]]), [0, 0], cache, logits="none", slots=[2]) is None and cache.host_lens[2] == 40
    out = dec.extend(rows([ids[2][0, 40:41]]), [0, 1], cache, logits="all", slots=[2])
    check(out, O.forward_multimodal(ids[2][:, :41], None, sd, oracle_cfg())[0][0, -1:], "a row that was passed over")


def test_what_extend_refuses(model):
    dec = model.model.decoder
    cache = dec.new_cache(2, 64)
    x = torch.zeros(70, dec.C, device="cuda", dtype=torch.bfloat16)
    for args, kw in [(([0, 1], ), {}), (([0, 1, 0],), {}), (([0, 40, 80],), {}), (([0, 1, 1],), dict(logits="last")), (([0, 1, 2],), dict(slots=[0, 0])),
                     (([0, 1],), dict(slots=[2])), (([0, 65, 66],), {})]:
        with pytest.raises(ValueError):
            dec.extend(x, args[0], cache, **kw)
    assert cache.host_lens == [0, 0]


@pytest.mark.parametrize("side", ["right", "left"])
def test_forward_behind_a_cache(sd, side):
    """A second turn with a padded mask, with an image, by embeddings, and what is refused."""
    model = _model(sd, tokenizer_padding_side=side)
    pixels, _ = tiny_inputs(1)
    a, b = _ids(30, 1), _ids(30, 2)
    turn = torch.cat([_ids(8, 5), _ids(8, 6)])
    mask = torch.ones(2, 8, dtype=torch.long)
    mask[1, (0 if side == "left" else 5):(3 if side == "left" else 8)] = 0
    cache = model(input_ids=torch.cat([a, b]), logits_to_keep=1, max_cache_len=700).past_key_values
    full = torch.cat([torch.ones(2, 30, dtype=torch.long), mask], 1)
    res = model(input_ids=turn, attention_mask=full, past_key_values=cache)
    assert res.logits.shape == (2, 8, TINY["vocab"]) and cache.host_lens == [38, 35] and res.past_key_values is cache
    for i, x in enumerate((a, b)):
        want = O.forward_multimodal(torch.cat([x, turn[i:i + 1, mask[i].bool()]], 1), None, sd, oracle_cfg())[0][0, 30:]
        got = res.logits[i][mask[i].bool().cuda()]
        check(got, want, f"second turn of sequence {i}")
        assert bool((res.logits[i][~mask[i].bool().cuda()] == 0).all())
    # third turn: an image and text for one sequence, by ids
    one = model(input_ids=a, logits_to_keep=1, max_cache_len=700).past_key_values
    ids = _ids(12, 7)
    ids[0, 4] = -200
    got = model(input_ids=ids, images=pixels[:1], past_key_values=one).logits
    want = O.forward_multimodal(torch.cat([a, ids], 1), pixels[:1], sd, oracle_cfg())[0]
    check(got[0], want[0, 30:], "a turn with an image")
    again = model(input_ids=a, logits_to_keep=1, max_cache_len=700).past_key_values
    hs = model(inputs_embeds=model.weights.llm.embed[turn[:1].cuda()], past_key_values=again, logits_to_keep=1, output_hidden_states=True)
    check(hs.logits[0], O.forward_multimodal(torch.cat([a, turn[:1]], 1), None, sd, oracle_cfg())[0][0, -1:], "by embeddings")
    assert len(hs.hidden_states) == TINY["layers"] + 1 and hs.hidden_states[0].shape == (1, 8, TINY["hidden"])
    for kw in (dict(input_ids=turn, labels=turn), dict(input_ids=turn[:, :3]), dict(), dict(input_ids=turn[:1], attention_mask=mask[:1, :5])):
        with pytest.raises(ValueError):
            model(past_key_values=again, **kw)


@pytest.mark.parametrize("scaling", [{"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32}, {"type": "linear", "factor": 2.5}])
def test_stretched_frequencies(sd, scaling, monkeypatch):
    """Prompt, chunk and decode step (every kernel that rotates) with a config's rope_scaling, against the oracle with the same angles and factor."""
    from omchat_b200 import rope

    def cos_sin(position_ids, cfg, dtype):
        turns, m = rope.frequencies(cfg.head_dim, cfg.rope_theta, scaling)
        ang = (position_ids.double()[..., None] * turns * 2 * math.pi).repeat(1, 1, 2)
        return (m * ang.cos()).to(dtype), (m * ang.sin()).to(dtype)

    monkeypatch.setattr(O, "rope_cos_sin", cos_sin)
    model, ids = _model(sd, rope_scaling=scaling), _ids(101, 4)
    want = O.forward_multimodal(ids, None, sd, oracle_cfg())[0]
    res = model(input_ids=ids[:, :60], max_cache_len=200)
    check(res.logits[0], want[0, :60], "prompt")
    check(model(input_ids=ids[:, 60:100], past_key_values=res.past_key_values).logits[0], want[0, 60:100], "chunk")
    check(model(input_ids=ids[:, 100:], past_key_values=res.past_key_values).logits[0], want[0, 100:], "decode step")
    plain = _model(sd)(input_ids=ids[:, :60]).logits
    assert (plain - res.logits).abs().max() > 0.05 * plain.abs().max()      # it does stretch


@pytest.mark.parametrize("slots,portion", [(3, 16), (6, 100)])
def test_prompts_in_portions_beside_decode_steps(model, sd, slots, portion):
    """Requests of different lengths through a small page pool, long prompts by portions between chunks of decode steps: the oracle's tokens for each."""
    from omchat_b200.serving import ContinuousBatcher
    g = torch.Generator().manual_seed(21)
    S = TINY["image_size"]
    reqs = []
    for n_text, n_img, max_new in [(20, 1, 9), (33, 0, 5), (70, 0, 12), (9, 0, 3), (25, 1, 7), (150, 0, 1), (16, 0, 10)]:
        ids = torch.randint(1, TINY["vocab"], (1, n_text + n_img), generator=g)
        for j in range(n_img):
            ids[0, 3 + 5 * j] = -200
        px = torch.randn(n_img, 3, S, S, generator=g).to(torch.bfloat16).float() if n_img else None
        reqs.append((ids, px, max_new))
    cb = ContinuousBatcher(model, slots=slots, max_ctx=512, total_pages=60, chunk=2, prefill_chunk=portion)
    free = len(cb.free_pages)
    rids = [cb.submit(ids, px, max_new_tokens=mn) for ids, px, mn in reqs]
    beside = 0
    while cb.queue or any(r is not None for r in cb.active):
        cb.step()
        filling = [r for r in cb.active if r is not None and r.embeds is not None]
        beside += bool(filling) and any(r is not None and r.embeds is None for r in cb.active)
        assert len(cb.free_pages) + sum(len(r.pages) for r in cb.active if r is not None) == free
    assert beside > 0 and len(cb.free_pages) == free
    for rid, (ids, px, mn) in zip(rids, reqs):
        want, step_logits = O.greedy_generate(ids, px, sd, oracle_cfg(), max_new_tokens=mn)
        assert len(cb.results[rid]) == mn
        _same_or_near_tie(cb.results[rid].tolist(), want, step_logits, f"request {rid}")
    with pytest.raises(ValueError):
        ContinuousBatcher(model, slots=2, max_ctx=64, prefill_chunk=0)


def test_sparse_layers():
    """The mixture-of-experts decoder goes on with a prompt as it takes the whole one (its own numbers: the routing of near ties is its own)."""
    from omchat_b200.config import OmChatQwen2MoeConfig
    from omchat_b200.model.moe import Qwen2MoeDecoder
    from omchat_b200.model.weights import random_init
    cfg = OmChatQwen2MoeConfig(num_hidden_layers=1, vocab_size=2048, mm_vision_tower=None)
    dec = Qwen2MoeDecoder(cfg, random_init(cfg, device="cuda", seed=3, vision=False).llm)
    n = 120
    emb = (torch.randn(n, 2048, generator=torch.Generator().manual_seed(4)) * 0.5).to(torch.bfloat16).cuda()
    pos, seq = torch.arange(n, dtype=torch.int32).cuda(), torch.zeros(n, dtype=torch.int32).cuda()
    want = dec.prefill(emb.clone(), pos, seq, [0, n], dec.new_cache(1, 200), logits="all")
    cache, got, first = dec.new_cache(1, 200), [], 0
    for m in (1, 40, 70, 9):
        got.append(dec.extend(emb[first:first + m], [0, m], cache, logits="all"))
        first += m
    cos = torch.nn.functional.cosine_similarity(torch.cat(got), want, dim=-1)
    assert int((cos < 0.999).sum()) <= 3 and cos.median() >= 0.9995
