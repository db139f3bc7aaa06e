"""Refusals and sizes of the mixture-of-experts entry points (no GPU call), and
the restatement that the GPU tests use against the oracle's decoder."""
import numpy as np
import pytest

import experts_ref as ref

ARG, WORKSPACE = -1, -6


@pytest.fixture(scope="module")
def lib():
    import mimg

    return mimg.load()


@pytest.fixture
def buf():
    a = np.zeros(1 << 16, np.uint8)
    base = (a.ctypes.data + 255) // 256 * 256
    return a, base


def test_plan_bytes(lib):
    f = lib.mimg_experts_plan_bytes
    assert f(1, 2, 8) == 4 * (64 + 64 + 2)
    assert f(0, 1, 1) == 4 * 64
    assert f(100, 3, 64) == 4 * (128 + 320 + 300)  # 65 places
    assert f(1 << 20, 16, 512) == 4 * (576 + 2 * (1 << 24))
    for bad in ((-1, 1, 1), ((1 << 20) + 1, 1, 1), (1 << 20, 17, 32), (1, 0, 4), (1, 33, 64), (1, 5, 4), (1, 1, 0), (1, 1, 513)):
        assert f(*bad) == 0, bad


def test_workspace_bytes_of_more_tokens_are_enough_for_fewer(lib):
    for f in (lambda t: lib.mimg_experts_route_workspace_bytes(t, 8), lambda t: lib.mimg_experts_route_workspace_bytes(t, 60),
              lambda t: lib.mimg_experts_route_workspace_bytes(t, 512), lambda t: lib.mimg_experts_plan_bytes(t, 2, 8),
              lambda t: lib.mimg_experts_swiglu_workspace_bytes(t, 2, 100, 512),
              lambda t: lib.mimg_experts_combine_workspace_bytes(t, 2, 100, 512)):
        n = [f(t) for t in range(1, 5000)]
        assert n == sorted(n)


def test_workspace_bytes(lib):
    a8 = lib.mimg_a8_workspace_bytes
    assert lib.mimg_experts_route_workspace_bytes(7, 60) >= 7 * 60 * 8
    assert lib.mimg_experts_swiglu_workspace_bytes(7, 2, 100, 512) >= a8(7, 512)
    assert lib.mimg_experts_combine_workspace_bytes(7, 2, 100, 512) >= a8(14, 512) + 14 * 100 * 4
    for bad in ((0, 2, 100, 512), (-1, 2, 100, 512), (7, 0, 100, 512), (7, 33, 100, 512), (7, 2, 0, 512), (7, 2, 100, 0)):
        assert lib.mimg_experts_swiglu_workspace_bytes(*bad) == 0 and lib.mimg_experts_combine_workspace_bytes(*bad) == 0
    for bad in ((0, 8), (-1, 8), (7, 0), (7, 513)):
        assert lib.mimg_experts_route_workspace_bytes(*bad) == 0


def test_plan_refusals(lib, buf):
    p = buf[1]
    call = lambda ids=p, T=4, top=2, n=8, plan=p + 4096, nb=4096: lib.mimg_experts_plan_dev(ids, T, top, n, plan, nb, None)  # noqa: E731
    for kw in (dict(T=-1), dict(T=(1 << 20) + 1), dict(top=0), dict(top=9), dict(top=33, n=64), dict(n=0), dict(n=513), dict(ids=None),
               dict(plan=None), dict(plan=p + 4098), dict(plan=p + 16)):
        assert call(**kw) == ARG, kw
    assert call(nb=4 * (64 + 64 + 8) - 1) == WORKSPACE


def test_route_refusals(lib, buf):
    p = buf[1]

    def call(x=p, r=p + 4096, T=4, k=64, n=8, top=2, ids=p + 8192, w=p + 9216, plan=p + 10240, nb=4096, ws=p + 16384, wsb=1 << 14):
        return lib.mimg_experts_route_dev(x, r, T, k, n, top, 1, ids, w, plan, nb, ws, wsb, None)

    for kw in (dict(T=-1), dict(k=0), dict(k=62), dict(k=-4), dict(k=(1 << 24) + 4), dict(n=0), dict(n=513), dict(top=0), dict(top=9),
               dict(x=None), dict(r=None), dict(ids=None), dict(w=None), dict(ws=None), dict(x=p + 4), dict(r=p + 4104),
               dict(ws=p + 16384 + 128), dict(plan=p + 10242)):
        assert call(**kw) == ARG, kw
    assert call(wsb=lib.mimg_experts_route_workspace_bytes(4, 8) - 1) == WORKSPACE
    assert call(nb=100) == WORKSPACE


def test_product_refusals_of_the_shape(lib, buf):
    p = buf[1]
    for T, top, n in ((-1, 2, 8), ((1 << 20) + 1, 1, 8), (4, 0, 8), (4, 9, 8), (4, 2, 0), (4, 2, 513)):
        assert lib.mimg_experts_swiglu_a8_dev(1, 1, n, p, T, top, p, 4096, p, p, 4096, None) == ARG
        assert lib.mimg_experts_combine_a8_dev(1, n, p, p, T, top, p, 4096, p, p, 4096, None) == ARG


def test_wrappers_raise(lib, buf):
    import mimg

    with pytest.raises(mimg.MimgError, match="experts_plan"):
        mimg.experts_plan_dev(buf[1], 4, 2, 513, buf[1], 4096, None)


@pytest.mark.parametrize("dt,k,block", [(66, 512, 256), (67, 768, 256), (64, 736, 32)])
def test_restated_products_are_the_oracles(oracle, dt, k, block):
    raw = oracle.synthetic_weight(dt, 40, k, seed=1, scale=1 / np.sqrt(k))
    x = np.random.default_rng(2).standard_normal((6, k), np.float32)
    w, d, m, dm = ref.parts(dt, raw, 40, k)
    mine = (w * d[..., None] - (0 if m is None else m * dm[..., None])).reshape(40, k)
    assert np.abs(oracle.dequantize(dt, raw, 40 * k).reshape(40, k) - mine).max() <= 2 * ref.EPS * np.abs(mine).max()
    y, bound = ref.product(x, raw, dt, 40, k)
    assert (np.abs(oracle.linear_a8(x, raw, dt, 40, k, block=block) - y) <= bound).all()


@pytest.mark.parametrize("lost", ["block", "plane", "mins"])
def test_the_bound_does_not_keep_a_lost_part(oracle, lost):
    """The products' bound is tight enough to notice one block, the low plane
    of the scales or the mins left out."""
    raw = oracle.synthetic_weight(66, 40, 1024, seed=3, scale=1 / 32)
    x = np.random.default_rng(4).standard_normal((6, 1024), np.float32)
    y, bound = ref.product(x, raw, 66, 40, 1024)
    b = raw.reshape(40, 4, 144).copy()
    if lost == "block":
        b[:, 2, :4] = 0
    elif lost == "mins":
        b[:, 1, 2:4] = 0
    else:
        b[:, 1, 4:8] &= 0xF8
    assert (np.abs(ref.product(x, b, 66, 40, 1024)[0] - y) > bound).mean() > 0.9


def test_config_of_a_file_with_experts():
    import decoder

    md = {"general.architecture": "llama", "llama.block_count": 2, "llama.embedding_length": 256, "llama.feed_forward_length": 512,
          "llama.attention.head_count": 4, "llama.context_length": 64, "llama.attention.layer_norm_rms_epsilon": 1e-5}
    assert "experts" not in decoder.config_from_metadata(md)
    assert "experts" not in decoder.config_from_metadata(dict(md, **{"llama.expert_count": 0}))
    c = decoder.config_from_metadata(dict(md, **{"llama.expert_count": 8, "llama.expert_used_count": 2}))
    assert (c["experts"], c["experts_used"]) == (8, 2) and decoder.Config(**c).experts_used == 2
    with pytest.raises(ValueError, match="expert_used_count"):
        decoder.config_from_metadata(dict(md, **{"llama.expert_count": 8}))
    with pytest.raises(ValueError, match="experts"):
        decoder.config_from_metadata({k.replace("llama", "qwen2"): "qwen2" if v == "llama" else v
                                      for k, v in dict(md, **{"llama.expert_count": 8, "llama.expert_used_count": 2}).items()})
    for n, used in ((4, 5), (4, 0), (64, 33), (513, 2), (-1, 1)):
        with pytest.raises(ValueError, match="experts"):
            decoder.Config(experts=n, experts_used=used)
