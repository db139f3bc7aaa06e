"""Models with experts from files: a container written, read, uploaded whole and
run gives the logits of the tensors themselves; a file with biases of its
experts is turned away."""
import struct

import numpy as np
import pytest

from test_gpu_serving_experts import gguf_bytes, model

pytestmark = pytest.mark.gpu


def metadata_of(cfg):
    return {"general.architecture": "llama", "llama.block_count": cfg["layers"], "llama.embedding_length": cfg["embed"],
            "llama.feed_forward_length": cfg["ffn"], "llama.attention.head_count": cfg["heads"],
            "llama.attention.head_count_kv": cfg["kv_heads"], "llama.context_length": cfg["context"],
            "llama.rope.dimension_count": cfg["rope_dims"], "llama.rope.freq_base": float(cfg["rope_theta"]),
            "llama.attention.layer_norm_rms_epsilon": float(np.float32(cfg["norm_eps"])),
            "llama.expert_count": cfg["experts"], "llama.expert_used_count": cfg["experts_used"]}


def up(n, a):
    return (n + a - 1) // a * a


def mim_bytes(md, tensors):
    """A container (version 0.2) of a weights and a metadata section."""
    items, pool = b"", b""
    for k, v in sorted(md.items()):
        key = len(pool), len(k)
        pool += k.encode()
        if isinstance(v, str):
            typ, cnt, payload = 5, len(v), len(pool)
            pool += v.encode()
        elif isinstance(v, float):
            typ, cnt, payload = 3, 0, struct.unpack("<Q", struct.pack("<d", v))[0]
        else:
            typ, cnt, payload = 1, 0, v
        items += struct.pack("<IIB3xIQ8x", *key, typ, cnt, payload)
    meta = b"MIMM" + struct.pack("<IQ", len(md), len(pool)) + items + pool
    weights, table, names = b"", b"", b""
    for name, (dt, shape, data) in sorted(tensors.items(), key=lambda t: t[0].encode()):
        raw = np.ascontiguousarray(data).tobytes()
        at = up(len(weights), 4096 if len(raw) >= 1 << 20 else 64)
        weights += bytes(at - len(weights)) + raw
        dims = [*shape, *[0] * (8 - len(shape))]
        table += struct.pack("<IIIB3x8QQQ", len(names), len(name), dt, len(shape), *dims, at, len(raw))
        names += name.encode()
    index_len = 16 + 2 * 64 + len(table) + len(names)
    meta_at = up(64 + index_len, 8)
    data_at = up(meta_at + len(meta), 4096)
    sections = b"".join(struct.pack("<IIQQB39x", kind, 0, off, n, 0) for kind, off, n in ((1, data_at, len(weights)), (2, meta_at, len(meta))))
    index = struct.pack("<IIQ", 2, len(tensors), len(names)) + sections + table + names
    out = b"MIM\0" + struct.pack("<HHII6Q", 0, 2, 0x0A0B0C0D, 4096, 64, index_len, data_at, len(weights), data_at + len(weights), 0) + index
    out += bytes(meta_at - len(out)) + meta
    return out + bytes(data_at - len(out)) + weights


def test_a_container_with_experts(gpu, tmp_path):
    import container
    import decoder

    cfg, tensors = model(experts=5, used=2, seed=7)
    path = tmp_path / "experts.mim"
    path.write_bytes(mim_bytes(metadata_of(cfg), tensors))
    f = container.MimFile(str(path))
    got_cfg = f.llama_config()
    assert got_cfg["experts"] == 5 and got_cfg["experts_used"] == 2
    sec, got = f.upload()
    assert sorted(got) == sorted(tensors)
    prompt = np.random.default_rng(8).integers(1, 400, 9)
    want = decoder.Decoder(cfg, tensors, max_rows=16).forward(prompt, np.arange(9))
    dec = decoder.Decoder(got_cfg, got, max_rows=16)
    assert np.array_equal(dec.forward(prompt, np.arange(9)).view(np.uint32), want.view(np.uint32))
    del dec, got
    sec.free()
    f.close()


@pytest.mark.parametrize("kind", ["gguf", "mim"])
def test_a_file_with_biases_of_its_experts(gpu, tmp_path, kind):
    import container
    import decoder
    import gguf

    cfg, tensors = model(seed=9)
    tensors["blk.1.ffn_up_exps.bias"] = (1, [cfg["experts"], cfg["ffn"]], np.ones((cfg["experts"], cfg["ffn"]), np.float32))
    path = tmp_path / kind
    path.write_bytes((gguf_bytes if kind == "gguf" else mim_bytes)(metadata_of(cfg), tensors))
    f = (gguf.GGUFFile if kind == "gguf" else container.MimFile)(str(path))
    sec, got = f.upload()
    with pytest.raises(gpu.NotHandled, match="ffn_up_exps.bias"):
        decoder.Decoder(cfg, got)
    del got
    sec.free()
    f.close()
