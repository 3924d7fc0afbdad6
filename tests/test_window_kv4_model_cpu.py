"""Host logic of the model with an attention window and with caches in 4 bits: which
options go together, what the steps refuse, which caches are made.  The layers are
replaced by a recorder, so no GPU is touched."""

import pytest
import torch

from qmoe import driver
from qmoe import model as qm
from qmoe.attention import KV4Cache, KVCache
from test_cache_model_cpu import _Causal, _tokens


def _config(extra=None, **kw):
    def load(cfg):
        for k, v in (extra or {}).items():
            setattr(cfg, k, v)
    return qm.Qwen3MoeInferenceConfig(qm.MoENeuronConfig(**kw), load_config=load)


def test_the_window_is_the_checkpoints_or_the_option():
    assert _config().window() == 0
    assert _config({"sliding_window": 4096}).window() == 0  # written in the config, not in use
    assert _config({"sliding_window": 4096, "use_sliding_window": False}).window() == 0
    assert _config({"sliding_window": 4096, "use_sliding_window": True}).window() == 4096
    assert _config({"sliding_window": None, "use_sliding_window": True}).window() == 0
    assert _config({"sliding_window": 4096, "use_sliding_window": True}, attention_window=0).window() == 0
    assert _config({"sliding_window": 4096, "use_sliding_window": True}, attention_window=100).window() == 100
    assert _config(attention_window=64).window() == 64
    with pytest.raises(ValueError, match="negative"):
        _config({"sliding_window": -5, "use_sliding_window": True}).window()


def test_options_that_do_not_go_together():
    for kw in (dict(kv_cache_bits=8), dict(kv_cache_bits=0), dict(attention_window=-1), dict(attention_sink=-1),
               dict(kv_cache_bits=4, kv_cache_budget=64)):
        with pytest.raises(ValueError, match="kv_cache_b|attention_"):
            qm.MoENeuronConfig(**kw)
    with pytest.raises(ValueError, match="window"):
        _config(attention_window=32, kv_cache_budget=64).window()


@pytest.mark.parametrize("kw", [dict(kv_cache_bits=4), dict(attention_window=5), dict(kv_cache_bits=4, attention_window=5,
                                                                                      attention_sink=2)], ids=str)
def test_steps_and_prefixes_refused(kw):
    m = _Causal(**kw)
    with pytest.raises(ValueError, match="prefix is shared"):
        m.share_prefix(_tokens(4))
    m.prefill(_tokens(2, 10), torch.tensor([10, 3]))
    n = len(m.calls)
    for call in (lambda: m.decode_step(_tokens(2), torch.tensor([21, 3])),
                 lambda: m.decode_step(_tokens(2), torch.tensor([4, -1])),
                 lambda: m.greedy_decode(_tokens(2), 12, use_graph=False),
                 lambda: m.greedy_decode(_tokens(2), 19, use_graph=False, positions=torch.tensor([3, 2]))):
        with pytest.raises(ValueError, match="steps at positions"):
            call()
    assert len(m.calls) == n and m.position == 10
    m.decode_step(_tokens(2), torch.tensor([20, 3]))
    assert m.calls[-1][3] == m.model.caches()[0].capacity  # the captured step's bucket


def test_caches_of_four_bits_and_of_bf16():
    m = _Causal(kv_cache_bits=4)
    for c in m.model.caches():
        assert isinstance(c, KV4Cache) and c.capacity == 21 and c.k.shape == (2, 1, 21, 8)
        assert c.rows is m.model.caches()[0].rows and len(c) == 2
    assert not m.model.plain_attention() and m._contiguous()
    w = _Causal(attention_window=5)
    assert type(w.model.caches()[0]) is KVCache and not w.model.plain_attention()
    assert w.model.layers[0].self_attn.window == 5
    assert _Causal().model.plain_attention()


def test_prompts_rows_are_kept_and_grow():
    c = _Causal(kv_cache_bits=4).model.caches()[0]
    cpu = torch.device("cpu")
    a = c.rows.of(2, 1, 8, 16, cpu)
    assert c.rows.of(2, 1, 5, 16, cpu) is a
    assert c.rows.of(2, 1, 9, 16, cpu).capacity == 9
    assert c.rows.of(3, 1, 4, 16, cpu).k.shape == (3, 1, 4, 16)


def test_driver_passes_the_options():
    made = {}

    class Stop(Exception):
        pass

    class Model:
        @staticmethod
        def get_neuron_config_cls():
            def config(**kw):
                made.update(kw)
                raise Stop
            return config

    for argv, want in (([], (16, None, 0)),
                       (["--kv-cache-bits", "4", "--attention-window", "0", "--attention-sink", "3"], (4, 0, 3))):
        with pytest.raises(Stop):
            driver.prepare_inference(Model, driver.parse_args(argv))
        assert (made["kv_cache_bits"], made["attention_window"], made["attention_sink"]) == want
