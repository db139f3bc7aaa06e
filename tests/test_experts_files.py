"""Files that ask for more of a mixture of experts than the decoder's graph has
are turned away, not run without it."""
import pytest

MD = {"general.architecture": "llama", "llama.block_count": 2, "llama.embedding_length": 256, "llama.feed_forward_length": 512,
      "llama.attention.head_count": 4, "llama.context_length": 64, "llama.attention.layer_norm_rms_epsilon": 1e-5,
      "llama.expert_count": 8, "llama.expert_used_count": 2}


@pytest.mark.parametrize("key,value", [("expert_shared_count", 1), ("expert_weights_norm", False), ("expert_weights_scale", 2.5),
                                       ("expert_gating_func", 2), ("expert_group_count", 4)])
def test_metadata_that_the_graph_does_not_have(key, value):
    import decoder

    with pytest.raises(ValueError, match=key):
        decoder.config_from_metadata(dict(MD, **{"llama." + key: value}))


@pytest.mark.parametrize("key,value", [("expert_shared_count", 0), ("expert_weights_norm", True), ("expert_weights_scale", 1.0),
                                       ("expert_weights_scale", 0.0), ("expert_gating_func", 1), ("expert_group_count", 1)])
def test_metadata_that_says_what_the_graph_does(key, value):
    import decoder

    assert decoder.config_from_metadata(dict(MD, **{"llama." + key: value}))["experts"] == 8


def test_dense_models_are_read_as_before():
    import decoder

    md = {k: v for k, v in MD.items() if "expert" not in k}
    assert decoder.config_from_metadata(dict(md, **{"llama.expert_gating_func": 2})) == decoder.config_from_metadata(md)


@pytest.mark.parametrize("name", ["ffn_gate_shexp.weight", "ffn_gate_inp.bias", "ffn_up_exps.bias", "exp_probs_b.bias"])
def test_tensors_that_the_graph_does_not_have(name):
    import decoder

    class Weight:
        def __init__(self, n, k):
            self.n, self.k, self.dt = n, k, 66

    d = object.__new__(decoder.Decoder)
    d.c = decoder.Config(layers=1, embed=256, ffn=512, heads=4, experts=8, experts_used=2)
    p = "blk.0."
    d.vec = {p + "ffn_gate_inp.weight": None}
    d.w = {f"{p}ffn_{s}_exps.weight": Weight(8 * n, k) for s, n, k in (("gate", 512, 256), ("up", 512, 256), ("down", 256, 512))}
    tensors = dict.fromkeys(d.w, (66, None, None))
    tensors[p + "ffn_gate_inp.weight"] = (1, [8, 256], None)
    d._check_experts(tensors)
    with pytest.raises(ValueError, match=name.replace(".", "[.]")):
        d._check_experts(dict(tensors, **{p + name: (1, [8], None)}))
