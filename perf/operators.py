"""Operators of a serving loop with an 8-bit key-value cache, as cases that can
be timed and checked: each in its plain form and through libmimg.

A case is a plain dict; `kind` names the operator:

  store      keys and values of new tokens into the 8-bit cache (one int8 scale
             for each block of 32 tokens and kv head), and the touched blocks
             read back: mimg.kv_store_q8_dev, mimg.kv_load_q8_dev
  attention  attention over that cache, prompts and decode batches:
             mimg.attention_q8_dev
  logprobs   log probabilities of given tokens, the entropy and the largest
             alternatives of each row of logits: mimg.logprobs_dev

`slots` sequences of `rows` new tokens each lie in a cache of slots * stride
entries, sequence i from entry i * stride on; stride is a multiple of 32.
Shapes are the two model shapes of the decode benchmarks (32 query and 8
key-value heads of 64 or 128, vocabulary 128256), the reference's 181-token
prompt, and odd sizes between.
"""
import math
import os
import random
import sys

import torch

own = False

BLOCK = 32  # cache entries that share a scale
FLOOR = 2.0 ** -96  # the smallest scale of a block that is not all zeros


# ---- the cases ---------------------------------------------------------------

def listed():
    return [
        # one decode step of eight sequences: a token appended to each, inside
        # a block whose scale may have to grow
        dict(kind="store", slots=8, stride=2048, base=1005, rows=1, kv_heads=8, d=128, name="append_8"),
        # the keys and values of a 512-token prompt into an empty cache
        dict(kind="store", slots=1, stride=768, base=0, rows=512, kv_heads=8, d=128, name="store_prompt_512"),
        # four prompts of 1000 tokens that go on behind 19 cached ones
        dict(kind="store", slots=4, stride=2048, base=19, rows=1000, kv_heads=8, d=64, name="store_4x1000_d64"),
        # one short chat, one token: launches and latency
        dict(kind="attention", slots=1, stride=256, base=180, rows=1, heads=32, kv_heads=8, d=64, name="decode_1x181_d64"),
        # a decode step of eight sequences deep into their contexts
        dict(kind="attention", slots=8, stride=2048, base=2020, rows=1, heads=32, kv_heads=8, d=128, name="decode_8x2048"),
        # a full serving batch
        dict(kind="attention", slots=64, stride=2048, base=2020, rows=1, heads=32, kv_heads=8, d=128, name="decode_64x2048"),
        # one token over a long document
        dict(kind="attention", slots=1, stride=131072, base=131000, rows=1, heads=32, kv_heads=8, d=128, name="decode_1x131072"),
        # the reference's 181-token prompt, three at once, odd heads a group
        dict(kind="attention", slots=3, stride=224, base=0, rows=181, heads=14, kv_heads=2, d=64, name="prompt_3x181_d64"),
        # a chunk of a long prompt over what is cached of it: the largest
        dict(kind="attention", slots=1, stride=8192, base=6100, rows=2048, heads=32, kv_heads=8, d=128, name="prompt_2048_at_6100"),
        # the token just sampled, with the twenty alternatives an API returns
        dict(kind="logprobs", rows=1, n=128256, ld=128256, top=20, masked=False, name="logprobs_1x128256"),
        # a prompt scored for its perplexity, five alternatives each
        dict(kind="logprobs", rows=512, n=128256, ld=128256, top=5, masked=False, name="logprobs_512x128256"),
        # a decode batch under a grammar, odd vocabulary: most logits -inf
        dict(kind="logprobs", rows=37, n=32003, ld=32003, top=8, masked=True, name="logprobs_37x32003_masked"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "attention", "attention", "logprobs"])
    if kind == "logprobs":
        n = _log(rng, 1000, 152064)
        rows = max(1, min(_log(rng, 1, 512), 512 * 128256 // n))
        return dict(kind=kind, rows=rows, n=n, ld=n + rng.choice([0, 0, 0, 1, 64]), top=rng.choice([0, 1, 5, 8, 20, 33]),
                    masked=rng.random() < 0.25)
    kv = rng.choice([1, 2, 4, 8])
    d = rng.choice([64, 64, 80, 128, 128, 128])
    if kind == "store":
        rows, slots = (1, _log(rng, 1, 64)) if rng.random() < 0.4 else (_log(rng, 2, 1024), rng.randint(1, 4))
        base = rng.choice([0, _log(rng, 1, 4096)])
        stride = (base + rows + 32 * slots + BLOCK - 1) // BLOCK * BLOCK
        return dict(kind=kind, slots=slots, stride=stride, base=base, rows=rows, kv_heads=kv, d=d)
    heads = kv * rng.choice([1, 2, 4, 4, 7, 8])
    if rng.random() < 0.5:  # a decode batch
        slots, rows = _log(rng, 1, 64), 1
        base = _log(rng, 16, max(17, min(131072, 131072 // slots)))
    else:
        slots, rows = rng.choice([1, 1, 2, 5]), _log(rng, 2, 1024)
        base = rng.choice([0, _log(rng, 1, 4096)])
        while slots * rows * (base + rows) * heads * d > 2048 * 7000 * 32 * 128:
            rows = (rows + 1) // 2
    return dict(kind=kind, slots=slots, stride=(base + rows + BLOCK - 1) // BLOCK * BLOCK, base=base, rows=rows,
                heads=heads, kv_heads=kv, d=d)


# ---- the sizes of a case -------------------------------------------------------

def _bases(c):
    """Tokens that each sequence has cached before the call: `base`, less some
    for the decode batches' later sequences (no two alike, the last idle)."""
    if c["kind"] == "store":  # the same place in a block for all, so that the touched blocks are as many
        return [c["base"] + BLOCK * (i * 5 % max(1, (c["stride"] - c["base"] - c["rows"]) // BLOCK + 1)) for i in range(c["slots"])]
    r = random.Random(c["base"] * 64 + c["slots"])
    return [c["base"] - (r.randrange(c["base"] // 4 + 1) if i else 0) for i in range(c["slots"])]


def _idle(c):
    """The last of a decode batch's sequences has no keys: a padded batch."""
    return c["kind"] == "attention" and c["rows"] == 1 and c["slots"] >= 8


def _touched(c):
    """Blocks that a sequence's new tokens reach, and the first one's filled entries."""
    off = c["base"] % BLOCK
    return (off + c["rows"] + BLOCK - 1) // BLOCK, off


# ---- inputs --------------------------------------------------------------------

class Draws:
    """Seeded values on the GPU; the same calls give the same values."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda", dtype=torch.float32)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda", dtype=torch.int64)


def _outliers(x):
    """A few channels of trained keys are several times the others."""
    x[..., 3::37] *= 4
    return x


def _encoded(x):
    """[kv_heads, L, d] -> int8 of the same shape and a scale for each 32 rows."""
    hk, length, d = x.shape
    b = x.reshape(hk, length // BLOCK, BLOCK * d)
    s = (b.abs().amax(-1) / 127).clamp_min(FLOOR)
    q = torch.round(b / s[..., None]).clamp(-127, 127).to(torch.int8)
    return q.reshape(hk, length, d), s


def _packed(kq, ks, vq, vs):
    """The library's layout of an 8-bit cache (include/mimg.h): a record of
    keys and values for each kv head and block, bytes value + 128, operands of
    the matrix cores in the order their lanes read them; then the scales."""
    hk, length, d = kq.shape
    nb, dp = length // BLOCK, (d + 63) // 64 * 64

    def padded(q):
        p = torch.full((hk, length, dp), 128, device=q.device, dtype=torch.uint8)
        p[..., :d] = (q.to(torch.int16) + 128).to(torch.uint8)
        return p

    k = padded(kq).reshape(hk, nb, 2, 16, dp // 64, 4, 16).permute(0, 1, 2, 4, 5, 3, 6).reshape(hk, nb, -1)
    v = padded(vq).reshape(hk, nb, 2, 4, 4, dp // 32, 2, 16).permute(0, 1, 5, 3, 7, 6, 2, 4).reshape(hk, nb, -1)
    meta = torch.zeros(hk, nb, 4, device=kq.device, dtype=torch.float32)
    meta[..., 0], meta[..., 1] = ks, vs
    return torch.cat([torch.cat([k, v], -1).reshape(-1), meta.reshape(-1).view(torch.uint8)])


def _cache(c, r):
    total = c["slots"] * c["stride"]
    kq, ks = _encoded(_outliers(r.normal(c["kv_heads"], total, c["d"])))
    vq, vs = _encoded(r.normal(c["kv_heads"], total, c["d"]))
    return kq, ks, vq, vs


def _prepare_store(c, seed):
    r = Draws(seed)
    kq, ks, vq, vs = _cache(c, r)
    new = (c["slots"] * c["rows"], c["kv_heads"], c["d"])
    k, v = _outliers(r.normal(*new)), r.normal(*new)
    at = torch.tensor([i * c["stride"] + b for i, b in enumerate(_bases(c))], device="cuda", dtype=torch.int64)
    m, off = _touched(c)
    index = (at[:, None] + torch.arange(c["rows"], device="cuda")).reshape(-1)
    read = ((at - off)[:, None] + torch.arange(m * BLOCK, device="cuda")).reshape(-1)
    back = (read.numel(), c["kv_heads"], c["d"])
    return dict(c, kq=kq, ks=ks, vq=vq, vs=vs, cache=_packed(kq, ks, vq, vs), k=k, v=v, index=index, read=read,
                k_out=torch.empty(back, device="cuda"), v_out=torch.empty(back, device="cuda"))


def _prepare_attention(c, seed):
    r = Draws(seed)
    kq, ks, vq, vs = _cache(c, r)
    q = r.normal(c["slots"] * c["rows"], c["heads"], c["d"])
    start = torch.arange(c["slots"], device="cuda", dtype=torch.int64) * c["stride"]
    end = start + torch.tensor(_bases(c), device="cuda", dtype=torch.int64)
    if _idle(c):
        end[-1] = start[-1] - 1
    rows = torch.arange(c["rows"], device="cuda", dtype=torch.int64)
    return dict(c, kq=kq, ks=ks, vq=vq, vs=vs, cache=_packed(kq, ks, vq, vs), q=q, out=torch.empty_like(q),
                start=start.repeat_interleave(c["rows"]), end=(end[:, None] + rows).reshape(-1))


def _prepare_logprobs(c, seed):
    r = Draws(seed)
    x = r.normal(c["rows"], c["ld"]) * 2.5
    # a model's favourites: up to eight tokens a row stand out
    x[:, :c["n"]].scatter_add_(1, r.ints(0, c["n"], c["rows"], 8), r.normal(c["rows"], 8).abs() * 6)
    if c["masked"]:  # a grammar leaves some fifty tokens of a row
        x[r.normal(c["rows"], c["ld"]) < math.sqrt(2 * math.log(max(2.0, c["n"] / 180)))] = -math.inf
        x[:, c["n"] // 2] = 1.0
    targets = r.ints(0, c["n"], c["rows"])
    if c["masked"]:
        targets[:] = c["n"] // 2
    if c["rows"] > 2:
        targets[-1] = -1  # a padded row
    top = (c["rows"], c["top"])
    return dict(c, x=x, targets=targets.to(torch.int32), lp=torch.empty(c["rows"], device="cuda"),
                entropy=torch.empty(c["rows"], device="cuda"), top_ids=torch.empty(top, device="cuda", dtype=torch.int32),
                top_lp=torch.empty(top, device="cuda"))


# ---- the plain forms -------------------------------------------------------------

def _plain_appended(s, q, scale, new):
    """The touched blocks [slots, kv_heads, m, 32, d] after the store, as values."""
    m, off = _touched(s)
    hk, d, slots, rows = s["kv_heads"], s["d"], s["slots"], s["rows"]
    blocks = (s["read"].reshape(slots, m, BLOCK)[..., 0] // BLOCK).reshape(-1)
    old_q = q.reshape(hk, -1, BLOCK, d)[:, blocks].reshape(hk, slots, m, BLOCK, d)
    old_s = scale[:, blocks].reshape(hk, slots, m)
    x = torch.zeros(hk, slots, m * BLOCK, d, device=q.device)
    x[:, :, off:off + rows] = new.reshape(slots, rows, hk, d).permute(2, 0, 1, 3)
    x = x.reshape(hk, slots, m, BLOCK, d)
    at = torch.arange(m * BLOCK, device=q.device).reshape(m, BLOCK)
    stored = (at >= off) & (at < off + rows)
    fresh = stored[:, 0]  # a block begins anew where its first entry is stored
    old_s = torch.where(fresh, torch.zeros_like(old_s), old_s)
    # scales rounded once, and the borders between two integers decided in 64 bits
    amax = x.abs().amax((-1, -2))
    s_new = torch.maximum(old_s, torch.where(amax > 0, (amax.double() / 127).float().clamp_min(FLOOR), amax))
    by = torch.where(s_new > 0, s_new, torch.ones_like(s_new)).double()[..., None, None]
    kept = old_q.double() * old_s.double()[..., None, None]
    out = torch.round(torch.where(stored[..., None], x.double(), kept) / by).float() * s_new[..., None, None]
    return out.reshape(hk, -1, d).transpose(0, 1).contiguous()


def _plain_store(s):
    return dict(k=_plain_appended(s, s["kq"], s["ks"], s["k"]), v=_plain_appended(s, s["vq"], s["vs"], s["v"]))


def _plain_attention(s):
    hk, d, slots, rows, n = s["kv_heads"], s["d"], s["slots"], s["rows"], s["stride"]
    g = s["heads"] // hk

    def values(q, scale):
        v = q.reshape(hk, -1, BLOCK, d).float() * scale[..., None, None]
        return v.reshape(hk, slots, n, d)

    q = s["q"].reshape(slots, rows, hk, g, d).permute(2, 0, 1, 3, 4).reshape(hk, slots, rows * g, d)
    p = torch.matmul(q, values(s["kq"], s["ks"]).transpose(2, 3)) * (1 / math.sqrt(d))
    at = torch.arange(n, device=q.device)
    seen = (at <= (s["end"] - s["start"]).reshape(slots, rows, 1)).repeat_interleave(g, 1)
    p.masked_fill_(~seen, -math.inf)
    p -= p.amax(-1, keepdim=True).clamp_min(-3e38)
    p.exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, values(s["vq"], s["vs"])) / torch.where(total > 0, total, torch.ones_like(total))
    return out.reshape(hk, slots, rows, g, d).permute(1, 2, 0, 3, 4).reshape(s["q"].shape)


def _plain_logprobs(s):
    x = s["x"][:, :s["n"]]
    best = x.amax(-1, keepdim=True)
    away = x - best
    e = torch.exp(away)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    entropy = log_total - torch.where(e > 0, e * away, torch.zeros_like(e)).sum(-1, keepdim=True) / total
    t = s["targets"].long()[:, None]
    given = (t >= 0) & (t < s["n"])
    lp = torch.gather(away, 1, t.clamp(0, s["n"] - 1)) - log_total
    out = dict(logprob=torch.where(given, lp, torch.zeros_like(lp))[:, 0], entropy=entropy[:, 0])
    if s["top"]:
        # one whole number orders the pairs (value, -index): ties to the lowest index
        bits = (x + 0.0).view(torch.int32)  # no negative zeros
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32
        ids = 0xFFFFFFFF - (torch.topk(order + (0xFFFFFFFF - torch.arange(s["n"], device=x.device)), s["top"], -1)[0] & 0xFFFFFFFF)
        out.update(top_ids=ids.to(torch.int32), top_logprobs=torch.gather(away, 1, ids) - log_total)
    return out


# ---- the framework's calls ---------------------------------------------------------

_mimg = None


def _library():
    """The library on the HIP runtime that torch has loaded."""
    global _mimg
    if _mimg is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mimir-model_amd"))
        os.environ.setdefault("MIMG_HIP_RUNTIME", os.path.join(os.path.dirname(torch.__file__), "lib", "libamdhip64.so"))
        import mimg

        mimg.init()
        _mimg = mimg
    return _mimg


def _workspace(s, nbytes):
    """A state's workspace, made at its first pass."""
    if "ws" not in s:
        s["ws"] = torch.empty(max(nbytes, 16), device="cuda", dtype=torch.uint8)
    return s["ws"].data_ptr(), s["ws"].numel()


def _own_store(s):
    lib, st, total = _library(), torch.cuda.current_stream().cuda_stream, s["slots"] * s["stride"]
    cache, hk, d = s["cache"].data_ptr(), s["kv_heads"], s["d"]
    lib.kv_store_q8_dev(s["k"].data_ptr(), s["v"].data_ptr(), s["index"].data_ptr(), s["index"].numel(), hk, d, total, cache, st)
    lib.kv_load_q8_dev(cache, s["read"].data_ptr(), s["read"].numel(), hk, d, total, s["k_out"].data_ptr(), s["v_out"].data_ptr(), st)
    return dict(k=s["k_out"], v=s["v_out"])


def _own_attention(s):
    lib, rows, total = _library(), s["slots"] * s["rows"], s["slots"] * s["stride"]
    ws = _workspace(s, lib.attention_q8_workspace_bytes(rows, s["heads"], s["kv_heads"], s["d"], s["stride"]) if "ws" not in s else 0)
    lib.attention_q8_dev(s["q"].data_ptr(), s["cache"].data_ptr(), s["end"].data_ptr(), s["start"].data_ptr(), rows, s["heads"],
                         s["kv_heads"], s["d"], total, s["stride"], s["out"].data_ptr(), *ws,
                         torch.cuda.current_stream().cuda_stream)
    return s["out"]


def _own_logprobs(s):
    lib, top = _library(), s["top"]
    ws = _workspace(s, lib.logprobs_workspace_bytes(s["rows"], s["n"], top) if "ws" not in s else 0)
    lib.logprobs_dev(s["x"].data_ptr(), s["rows"], s["n"], s["ld"], s["targets"].data_ptr(), top, s["lp"].data_ptr(),
                     s["entropy"].data_ptr(), s["top_ids"].data_ptr() if top else None, s["top_lp"].data_ptr() if top else None,
                     *ws, torch.cuda.current_stream().cuda_stream)
    out = dict(logprob=s["lp"], entropy=s["entropy"])
    return dict(out, top_ids=s["top_ids"], top_logprobs=s["top_lp"]) if top else out


# ---- in 64 bits, from the definitions ------------------------------------------------

def _exact_store(c, seed):
    """Token by token position: what each entry of a touched block stands for."""
    s = _prepare_store(c, seed)
    m, off = _touched(c)
    filled = off + c["rows"]
    out = {}
    for name, q, scale, new in (("k", s["kq"], s["ks"], s["k"]), ("v", s["vq"], s["vs"], s["v"])):
        new = new.double().reshape(c["slots"], c["rows"], c["kv_heads"], c["d"])
        back = torch.empty(c["slots"], m, BLOCK, c["kv_heads"], c["d"], device="cuda", dtype=torch.float64)
        for j in range(m):
            lo, hi = max(off, j * BLOCK), min(filled, (j + 1) * BLOCK)
            first = s["read"].reshape(c["slots"], m, BLOCK)[:, j, 0]
            part = new[:, lo - off:hi - off]
            largest = part.abs().amax((1, 3))  # [slots, kv_heads]
            # a scale is a float32: 127ths of the largest value, rounded
            step = torch.clamp((largest / 127).float(), min=FLOOR).double() * (largest > 0)
            block = torch.zeros(c["slots"], BLOCK, c["kv_heads"], c["d"], device="cuda", dtype=torch.float64)
            if lo > j * BLOCK:  # not from the block's first entry on: the others stay
                was = scale[:, first // BLOCK].T.double()
                step = torch.maximum(step, was)
                rows = first[:, None] + torch.arange(BLOCK, device="cuda")
                block = q.double().transpose(0, 1)[rows] * was[:, None, :, None]
            block[:, lo - j * BLOCK:hi - j * BLOCK] = part
            divide = torch.where(step > 0, step, torch.ones_like(step))[:, None, :, None]
            back[:, j] = torch.round(block / divide) * step[:, None, :, None]
        out[name] = back.reshape(-1, c["kv_heads"], c["d"])
    return out


def _exact_attention(c, seed):
    s = _prepare_attention(c, seed)
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    for i in range(c["slots"]):
        rows, keys = slice(i * c["rows"], (i + 1) * c["rows"]), slice(i * c["stride"], (i + 1) * c["stride"])
        end = s["end"][rows] - s["start"][rows]
        if int(end.max()) < 0:
            continue
        hidden = torch.arange(c["stride"], device="cuda")[None, :] > end[:, None]
        for h in range(c["kv_heads"]):
            block = slice(i * c["stride"] // BLOCK, (i + 1) * c["stride"] // BLOCK)
            k = s["kq"][h, keys].double() * s["ks"][h, block].double().repeat_interleave(BLOCK)[:, None]
            v = s["vq"][h, keys].double() * s["vs"][h, block].double().repeat_interleave(BLOCK)[:, None]
            for g in range(c["heads"] // c["kv_heads"]):
                head = h * (c["heads"] // c["kv_heads"]) + g
                score = (s["q"][rows, head].double() @ k.T / math.sqrt(c["d"])).masked_fill(hidden, -math.inf)
                out[rows, head] = torch.softmax(score, -1) @ v
    return out


def _exact_logprobs(c, seed):
    s = _prepare_logprobs(c, seed)
    x = s["x"][:, :c["n"]]
    p = torch.log_softmax(x.double(), -1)
    t = s["targets"].long()
    lp = p[torch.arange(c["rows"], device="cuda"), t.clamp_min(0)]
    lp[t < 0] = 0
    out = dict(logprob=lp, entropy=torch.special.entr(p.exp()).sum(-1))
    if c["top"]:
        ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :c["top"]]
        out.update(top_ids=ids.to(torch.int32), top_logprobs=torch.gather(p, 1, ids))
    return out


# ---- the interface ---------------------------------------------------------------------

def prepare(case, seed):
    return {"store": _prepare_store, "attention": _prepare_attention, "logprobs": _prepare_logprobs}[case["kind"]](case, seed)


def run(state):
    if own:
        return {"store": _own_store, "attention": _own_attention, "logprobs": _own_logprobs}[state["kind"]](state)
    return {"store": _plain_store, "attention": _plain_attention, "logprobs": _plain_logprobs}[state["kind"]](state)


def exact(case, seed):
    return {"store": _exact_store, "attention": _exact_attention, "logprobs": _exact_logprobs}[case["kind"]](case, seed)


def work(case):
    """Inputs read and outputs written once; two operations for each product."""
    c = case
    if c["kind"] == "logprobs":
        return dict(bytes=4 * c["rows"] * c["n"] + c["rows"] * (12 + 8 * c["top"]), flops=4 * c["rows"] * c["n"])
    if c["kind"] == "store":
        m, off = _touched(c)
        new, row = c["slots"] * c["rows"], 2 * c["kv_heads"] * c["d"]
        held = c["slots"] * (BLOCK if off else 0)  # entries of the block that is continued
        return dict(bytes=row * (4 * new + new + held + 4 * c["slots"] * m * BLOCK), flops=2 * row * new)
    d, lens = c["d"], [b + c["rows"] for b in _bases(c)]
    pairs = [sum(range(b + 1, b + c["rows"] + 1)) for b in _bases(c)]
    if _idle(c):
        lens, pairs = lens[:-1], pairs[:-1]
    return dict(bytes=2 * c["kv_heads"] * sum(lens) * (d + 8 / BLOCK) + 8 * c["slots"] * c["rows"] * c["heads"] * d,
                flops=4 * sum(pairs) * c["heads"] * d)
