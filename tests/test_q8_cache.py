"""The 8-bit cache's layout and the refusals of its operators and of the log
probabilities, without a GPU: every check of arguments comes before the first
GPU call."""
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest

import mimg
import q8_ref

ARG, WS = -1, -6
P = 1 << 20  # an address that no call may read


def layout_byte(e, i, dp):
    """include/mimg.h's formulas."""
    key = (((e // 16) * (dp // 64) + i // 64) * 64 + (i // 16 % 4) * 16 + e % 16) * 16 + i % 16
    value = 32 * dp + ((i // 32) * 64 + (e // 4 % 4) * 16 + i % 16) * 16 + (i // 16 % 2) * 8 + (e // 16) * 4 + e % 4
    return key, value


@pytest.mark.parametrize("hk,context,d", [(1, 32, 64), (2, 70, 128), (3, 33, 8), (1, 100, 80), (2, 64, 192), (1, 40, 256)])
def test_pack_follows_the_header(hk, context, d):
    rng = np.random.default_rng(d + context)
    nb, dp = (context + 31) // 32, (d + 63) // 64 * 64
    k, v = (rng.integers(-127, 128, (hk, context, d)).astype(np.int8) for _ in range(2))
    ks, vs = (rng.random((hk, nb)).astype(np.float32) for _ in range(2))
    bad = rng.integers(0, 1 << 32, (hk, nb), dtype=np.uint32)
    raw = mimg.pack_cache_q8(k, ks, v, vs, bad)
    assert raw.size == mimg.cache_q8_bytes(hk, context, d)
    for h in range(hk):
        for j in range(context):
            rec = raw[(h * nb + j // 32) * 64 * dp:]
            for i in range(0, d, 3):
                kb, vb = layout_byte(j % 32, i, dp)
                assert int(rec[kb]) - 128 == k[h, j, i] and int(rec[vb]) - 128 == v[h, j, i]
    back = mimg.unpack_cache_q8(raw, hk, context, d)
    for got, want in zip(back, (k, ks, v, vs, bad)):
        assert np.array_equal(got, want)


def test_layout_is_a_bijection():
    for dp in (64, 128, 192, 256):
        seen = sorted(b for e in range(32) for i in range(dp) for b in layout_byte(e, i, dp))
        assert seen == list(range(64 * dp))


def test_sizes():
    assert mimg.cache_q8_bytes(8, 8192, 128) == 8 * 256 * (64 * 128 + 16)
    assert mimg.cache_q8_bytes(1, 1 << 30, 256) == (1 << 25) * (64 * 256 + 16)  # past 32 bits
    for hk, c, d in ((0, 32, 64), (1, 0, 64), (1, 32, 0), (1, 32, 12), (1, 32, 264), (1, (1 << 30) + 1, 64), (16385, 32, 64),
                     (-1, 32, 64), (1, -5, 64)):
        assert mimg.cache_q8_bytes(hk, c, d) == 0
    assert mimg.attention_q8_workspace_bytes(0, 8, 8, 64, 100) == 0
    assert mimg.attention_q8_workspace_bytes(1, 32, 8, 128, 1 << 20) > 0
    assert mimg.attention_q8_workspace_bytes(1, 32, 7, 128, 1 << 20) == 0
    assert mimg.logprobs_workspace_bytes(1, 128256, 20) > 0
    assert mimg.logprobs_workspace_bytes(1, 10, 11) == 0 and mimg.logprobs_workspace_bytes(1, (1 << 21) + 1, 1) == 0


def refused(code, text, fn, *args):
    """In a thread of its own: the library keeps the last error by thread."""
    with ThreadPoolExecutor(1) as ex, pytest.raises(mimg.MimgError) as e:
        ex.submit(fn, *args).result()
    assert e.value.code == code, e.value
    assert text in str(e.value)


@pytest.mark.parametrize("change", [dict(T=-1), dict(T=65536), dict(hk=0), dict(hk=16385), dict(d=0), dict(d=4), dict(d=12),
                                    dict(d=264), dict(context=0), dict(context=(1 << 30) + 1), dict(cache=P + 8),
                                    dict(cache=0), dict(k=0), dict(v=0), dict(index=0)])
def test_store_and_load_refuse(change):
    a = dict(T=3, hk=2, d=64, context=100, cache=P, k=P, v=P, index=P)
    a.update(change)
    text = "16-byte aligned" if a["cache"] == P + 8 else "null" if 0 in (a["cache"], a["k"], a["v"], a["index"]) else "kv_"
    refused(ARG, text, mimg.kv_store_q8_dev, a["k"], a["v"], a["index"], a["T"], a["hk"], a["d"], a["context"], a["cache"], 0)
    refused(ARG, text, mimg.kv_load_q8_dev, a["cache"], a["index"], a["T"], a["hk"], a["d"], a["context"], a["k"], a["v"], 0)
    if text == "kv_":
        text = "rope_kv_q8"
    refused(ARG, text, mimg.rope_kv_q8_dev, P, a["k"], a["v"], P, a["index"], P, a["T"], 4, a["hk"], a["d"], 8, 0, a["context"],
            a["cache"], 0)


@pytest.mark.parametrize("change", [dict(H=0), dict(H=16385), dict(rotary=0), dict(rotary=7), dict(rotary=66), dict(q=0),
                                    dict(pos=0), dict(freq=0)])
def test_rope_refuses(change):
    a = dict(H=4, rotary=64, q=P, pos=P, freq=P)
    a.update(change)
    refused(ARG, "null" if 0 in (a["q"], a["pos"], a["freq"]) else "rope_kv_q8", mimg.rope_kv_q8_dev, a["q"], P, P, a["pos"], P,
            a["freq"], 3, a["H"], 2, 64, a["rotary"], 1, 100, P, 0)


@pytest.mark.parametrize("change", [dict(T=-1), dict(T=65536), dict(H=0), dict(H=7), dict(H=16386), dict(hk=0), dict(hk=-2),
                                    dict(d=0), dict(d=20), dict(d=264), dict(context=0), dict(maxk=0), dict(maxk=(1 << 30) + 1),
                                    dict(q=0), dict(cache=0), dict(cache=P + 1), dict(kend=0), dict(out=0), dict(ws=0),
                                    dict(ws=P + 8), dict(wsb=-1), dict(out=P + 64)])
def test_attention_refuses(change):
    a = dict(T=2, H=8, hk=2, d=64, context=1 << 16, maxk=1 << 16, q=P, cache=P << 8, kend=P, out=P << 4, ws=P << 6, wsb=0)
    a.update(change)
    need = mimg.attention_q8_workspace_bytes(2, 8, 2, 64, 1 << 16)
    assert need > 0
    code = WS if a["wsb"] < 0 else ARG
    refused(code, "attention_q8" if code == WS else "", mimg.attention_q8_dev, a["q"], a["cache"], a["kend"], None, a["T"], a["H"],
            a["hk"], a["d"], a["context"], a["maxk"], a["out"], a["ws"], need + a["wsb"], 0)


@pytest.mark.parametrize("change", [dict(rows=-1), dict(rows=(1 << 22) + 1), dict(n=0), dict(n=(1 << 21) + 1), dict(ld=99),
                                    dict(ld=(1 << 31) + 1), dict(top=-1), dict(top=65), dict(n=3, top=4), dict(x=0), dict(ws=0),
                                    dict(ws=P + 4), dict(wsb=-1), dict(targets=None),
                                    dict(lp=None, ent=None, ids=None, tlp=None), dict(lp=None, ent=None, top=0)])
def test_logprobs_refuse(change):
    a = dict(rows=2, n=100, ld=100, top=5, x=P, targets=P, lp=P, ent=P, ids=P, tlp=P, ws=P, wsb=0)
    a.update(change)
    need = mimg.logprobs_workspace_bytes(2, 100, 5)
    refused(WS if a["wsb"] < 0 else ARG, "", mimg.logprobs_dev, a["x"], a["rows"], a["n"], a["ld"], a["targets"], a["top"], a["lp"],
            a["ent"], a["ids"], a["tlp"], a["ws"], need + a["wsb"], 0)


def test_oracle_store_rules():
    """The restatement itself: a block begins anew with its first entry, a
    grown scale requantizes, of two rows with one index the later stays."""
    c = q8_ref.Cache(1, 64, 8)
    one = lambda x: np.full((1, 1, 8), x, np.float32)  # noqa: E731
    c.store(one(1.0), one(-1.0), [0])
    assert c.ks[0, 0] == np.float32(1 / 127) and c.k[0, 0, 0] == 127 and c.v[0, 0, 0] == -127
    c.store(one(2.0), one(0.5), [1])
    assert c.ks[0, 0] == np.float32(2 / 127) and list(c.k[0, :2, 0]) == [64, 127] and list(c.v[0, :2, 0]) == [-127, 64]
    c.store(np.concatenate([one(3.0), one(4.0)]), np.concatenate([one(1.0), one(1.0)]), [0, 0])
    assert c.k[0, 0, 0] == 127 and c.ks[0, 0] == np.float32(4 / 127) and not c.k[0, 1:].any()
    c.store(one(np.nan), one(1.0), [5])
    assert c.bad[0, 0] == 1 << 5 and np.isnan(c.values()[0][0, 5]).all() and not np.isnan(c.values()[0][0, 4]).any()
