"""The attention window's options: what a checkpoint's config means, when a window
hides nothing, and what is refused when.  The layers are replaced by a recorder, so
no GPU is touched."""

import json

import pytest

from qmoe import model as qm


def _config(extra=None, **kw):
    def load(cfg):
        for k, v in (extra or {}).items():
            setattr(cfg, k, v)
    return qm.Qwen3MoeInferenceConfig(qm.MoENeuronConfig(**kw), load_config=load)


# ------------------------------------------------------------------ the checkpoint's config
def test_a_window_in_use_without_a_length_has_the_published_default(tmp_path):
    """The published config class has 4096 for a key that is absent, and no window for
    one that is null."""
    assert _config({"use_sliding_window": True}).window() == 4096
    assert _config({"use_sliding_window": True, "sliding_window": None}).window() == 0
    assert _config({"use_sliding_window": False}).window() == 0
    assert _config({"use_sliding_window": True}, attention_window=0).window() == 0
    assert _config({"use_sliding_window": True}, attention_window=100).window() == 100
    for written, want in (({"use_sliding_window": True}, 4096), ({"use_sliding_window": True, "sliding_window": None}, 0),
                          ({"use_sliding_window": True, "sliding_window": 77}, 77), ({}, 0)):
        (tmp_path / "config.json").write_text(json.dumps(written))
        config = qm.Qwen3MoeInferenceConfig(qm.MoENeuronConfig(), qm.load_pretrained_config(str(tmp_path)))
        assert config.window() == want, written


@pytest.mark.parametrize("kw", [{}, {"use_sliding_window": True}, {"use_sliding_window": True, "sliding_window": None},
                                {"use_sliding_window": True, "sliding_window": 77}, {"sliding_window": 77}], ids=str)
def test_the_window_of_the_published_config_class(kw):
    published = pytest.importorskip("transformers").Qwen3MoeConfig(**kw)
    assert _config(kw).window() == (published.sliding_window or 0)
