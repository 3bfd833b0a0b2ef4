"""Frequencies of rotary positions, plain and stretched (rope.frequencies), and how a config.json brings them in."""
import json
import math

import pytest
import torch

from omchat_b200 import rope
from omchat_b200.config import OmChatQwen2Config
from omchat_b200.model.checkpoint import config_from_dict, save_checkpoint


def _plain(n, theta):
    return torch.tensor([theta ** (-2.0 * i / n) for i in range(n // 2)], dtype=torch.float64)


@pytest.mark.parametrize("n,theta", [(128, 1e6), (64, 1e4), (2, 10.0), (0, 1e4)])
def test_plain_and_linear(n, theta):
    t, m = rope.frequencies(n, theta)
    assert t.dtype == torch.float64 and m == 1.0 and torch.allclose(t * 2 * math.pi, _plain(n, theta), rtol=1e-14, atol=0)
    t, m = rope.frequencies(n, theta, {"type": "linear", "factor": 8})
    assert m == 1.0 and torch.allclose(t * 16 * math.pi, _plain(n, theta), rtol=1e-14, atol=0)
    assert torch.equal(rope.frequencies(n, theta, {"rope_type": "default"})[0], rope.frequencies(n, theta)[0])


def test_yarn():
    n, theta, span, s = 128, 1e6, 32768, 4.0
    t, m = rope.frequencies(n, theta, {"rope_type": "yarn", "factor": s, "original_max_position_embeddings": span})
    plain = _plain(n, theta)
    made = span * plain / (2 * math.pi)                      # turns over the trained span
    share = t * 2 * math.pi / plain                          # 1: as it was, 1 / s: divided
    assert m == pytest.approx(0.1 * math.log(4) + 1, rel=1e-15)
    # the ramp's ends are whole pairs, just outside the borders
    low = math.floor(n * math.log(span / (32 * 2 * math.pi)) / (2 * math.log(theta)))
    high = math.ceil(n * math.log(span / (2 * math.pi)) / (2 * math.log(theta)))
    assert (made[:low + 1] >= 32).all() and torch.allclose(share[:low + 1], torch.ones(low + 1, dtype=torch.float64), rtol=1e-14)
    assert (made[high:] <= 1).all() and torch.allclose(share[high:], torch.full((n // 2 - high,), 1 / s, dtype=torch.float64), rtol=1e-14)
    steps = share[low:high + 1].diff()
    assert (steps < 0).all() and torch.allclose(steps, steps[:1].expand_as(steps), rtol=1e-10)
    assert rope.frequencies(n, theta, {"type": "yarn", "factor": s, "original_max_position_embeddings": span, "attention_factor": 1.5})[1] == 1.5
    m = rope.frequencies(n, theta, {"type": "yarn", "factor": 40, "original_max_position_embeddings": 4096, "mscale": 0.7, "mscale_all_dim": 1.4})[1]
    assert m == pytest.approx((0.07 * math.log(40) + 1) / (0.14 * math.log(40) + 1), rel=1e-14)


def test_llama3():
    span, s = 8192, 8.0
    kind = {"rope_type": "llama3", "factor": s, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": span}
    t, m = rope.frequencies(128, 5e5, kind)
    plain, w = _plain(128, 5e5), t * 2 * math.pi
    wave = 2 * math.pi / plain
    for i in range(64):
        if wave[i] < span / 4:
            want = plain[i]
        elif wave[i] > span:
            want = plain[i] / s
        else:
            smooth = (span / wave[i] - 1.0) / 3.0
            want = (1 - smooth) * plain[i] / s + smooth * plain[i]
        assert float(w[i]) == pytest.approx(float(want), rel=1e-13)
    assert m == 1.0


@pytest.mark.parametrize("bad,error", [({"type": "yarn", "factor": 4.0}, ValueError), ({"type": "linear"}, ValueError), ({"type": "longrope"}, NotImplementedError),
                                       ({"rope_type": "dynamic", "factor": 2.0}, NotImplementedError), ({"type": "llama3", "factor": 8.0}, ValueError)])
def test_what_is_refused(bad, error):
    with pytest.raises(error):
        rope.frequencies(128, 1e6, bad)
    with pytest.raises(ValueError):
        rope.frequencies(7, 1e6)


@pytest.mark.parametrize("hub", [False, True])
def test_config_json(tmp_path, hub):
    scaling = {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    c = OmChatQwen2Config(num_hidden_layers=1, rope_scaling=scaling)
    save_checkpoint({"model.norm.weight": torch.zeros(4)}, c, str(tmp_path), hub_layout=hub)
    d = json.load(open(tmp_path / "config.json"))
    assert config_from_dict(d).rope_scaling == scaling
    assert config_from_dict({"hidden_size": 256}).rope_scaling is None
    # base and scaling in one dictionary
    new = config_from_dict({"rope_parameters": {"rope_theta": 5e5, "rope_type": "linear", "factor": 2.0}})
    assert new.rope_theta == 5e5 and new.rope_scaling == {"rope_type": "linear", "factor": 2.0}
    assert config_from_dict({"rope_parameters": {"rope_theta": 1e4, "rope_type": "default"}}).rope_scaling is None


@pytest.mark.parametrize("d", [{"rope_scaling": {"type": "dynamic", "factor": 2.0}}, {"rope_parameters": {"rope_type": "longrope", "rope_theta": 1e4}}])
def test_kinds_that_are_not_built_change_nothing(d):
    with pytest.warns(RuntimeWarning, match="not built"):
        assert config_from_dict(d).rope_scaling is None


def test_the_trained_span_is_that_of_the_config():
    given = {"type": "yarn", "factor": 2.0}
    assert config_from_dict({"max_position_embeddings": 4096, "rope_scaling": given}).rope_scaling == {**given, "original_max_position_embeddings": 4096}
    own = {**given, "original_max_position_embeddings": 512}
    assert config_from_dict({"max_position_embeddings": 4096, "rope_scaling": own}).rope_scaling == own


def test_auto_config_keeps_it():
    import omchat_b200.hf as H
    scaling = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    assert H.OmChatQwen2Config(rope_scaling=dict(scaling)).to_native().rope_scaling == scaling
    assert H.OmChatQwen2Config().to_native().rope_scaling is None
