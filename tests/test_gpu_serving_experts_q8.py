"""The decoder with Q8_0 experts against the CPU restatement of the graph, their
products restated in the kernels' own order: exact integer sums of the blocks of
32, one float32 fma a block. So the only differences are those of the K-quant
experts (float64 sums of rms_norm and of the router, the weights'
exponentials), and the same 1e-3 of the largest logit is allowed: one 8-bit
integer that moves over a rounding border."""
import numpy as np
import pytest

import experts_ref as ref
import fixture_models as fm
import llama_ref
from test_gpu_serving_experts import Q4_K, Q6_K, Q8_0, RefDecoder, model

pytestmark = pytest.mark.gpu


class InOrder(RefDecoder):
    def product(self, x, name, e):
        dt, (_, n, k), w = self.m.t[name]
        if dt != Q8_0:
            return super().product(x, name, e)
        raw = np.asarray(w).reshape(-1, n * k // 32 * 34)[e]
        q, dx = ref.acts(x, 32)
        w, d, _, _ = ref.parts(dt, raw, n, k)
        sums = np.einsum("rbk,nbk->rnb", q, w)
        scale = (d.astype(np.float32)[None] * dx.astype(np.float32)[:, None]).astype(np.float64)
        y = np.zeros((x.shape[0], n), np.float32)
        for b in range(k // 32):  # (a product is exact in float64; the sum is rounded there first)
            y = (y + sums[..., b] * scale[..., b]).astype(np.float32)
        return y


@pytest.mark.parametrize("kw", [dict(experts=6, used=2, gate=Q8_0, down=Q8_0, ffn=288), dict(experts=9, used=3, gate=Q8_0, down=Q8_0, ffn=96),
                                dict(experts=20, used=4, gate=Q8_0, down=Q6_K), dict(experts=8, used=2, gate=Q4_K, down=Q8_0)])
def test_steps_match_the_restatement(gpu, oracle, kw):
    import decoder

    cfg, tensors = model(seed=11, **kw)
    dec = decoder.Decoder(cfg, tensors, max_rows=32)
    refd = InOrder(llama_ref.Model(cfg, tensors))
    prompt = np.random.default_rng(12).integers(1, 400, 23)
    want = refd.forward(prompt, np.arange(23))
    assert len(np.unique(np.stack(refd.chosen))) == cfg["experts"]
    ok, worst, allowed = fm.near(dec.forward(prompt, np.arange(23)), want, 1e-3)
    assert ok, f"prompt logits: {worst} > {allowed}"
    for i in range(4):
        tok = int(np.argmax(want[-1]))
        want = refd.forward([tok], [23 + i])
        ok, worst, allowed = fm.near(dec.forward([tok], [23 + i]), want, 1e-3)
        assert ok, f"step {i}: {worst} > {allowed}"
