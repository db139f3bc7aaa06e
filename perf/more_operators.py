"""Operators of a feed-forward layer that is a mixture of experts with
block-quantized weights, as cases that can be timed and checked: each in its
plain form and through libmimg.

A case is a plain dict; `kind` names the operator:

  route    the router: each token's logits over the experts, the largest few
           with their weights, and the plan that puts the chosen (token,
           choice) pairs in order by expert: mimg.experts_route_dev
  gate_up  the chosen experts' gate and up products on 8-bit activations and
           swiglu of the two: mimg.experts_swiglu_a8_dev
  down     the chosen experts' down products on 8-bit activations, summed over
           a token's choices with the router's weights:
           mimg.experts_combine_a8_dev

An expert's weights are [hidden, width] (gate, up) and [width, hidden] (down)
matrices in the blocks of Q4_K, Q6_K or Q8_0, the experts of a layer one
behind the other. Activations are quantized in blocks of 256 for Q4_K and
Q6_K and of 32 for Q8_0. Shapes are the feed-forward sizes of the decode
benchmarks (4096 x 14336, 2048 x 8192 cut in eight), the reference's 181-token
prompt, and odd sizes between.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"q4_k": (66, 256, 144), "q6_k": (67, 256, 210), "q8_0": (64, 32, 34)}  # id, weights and bytes of a block


# ---- the cases ---------------------------------------------------------------

def listed():
    return [
        # the token of a decode step, eight experts
        dict(kind="route", tokens=1, width=4096, experts=8, top=2, normalize=True, name="route_1_of_8"),
        # the reference's prompt, an odd number of experts, weights that are not normalized again
        dict(kind="route", tokens=181, width=2048, experts=60, top=4, normalize=False, name="route_181_of_60"),
        # a chunk of a long prompt over many experts
        dict(kind="route", tokens=2048, width=4096, experts=128, top=8, normalize=True, name="route_2048_of_128"),
        # a decode step of one sequence, large experts
        dict(kind="gate_up", tokens=1, width=4096, hidden=14336, experts=8, top=2, type="q4_k", padded=0, name="gate_up_1_of_8"),
        # a decode step of eight sequences, many small experts
        dict(kind="gate_up", tokens=8, width=2048, hidden=1024, experts=64, top=8, type="q4_k", padded=0, name="gate_up_8_of_64"),
        # a serving batch, where every large expert has a few tokens
        dict(kind="gate_up", tokens=64, width=4096, hidden=14336, experts=8, top=2, type="q4_k", padded=0, name="gate_up_64_of_8"),
        # the reference's prompt in 8 bits, a hidden size that is no multiple of 256
        dict(kind="gate_up", tokens=181, width=2048, hidden=1408, experts=60, top=4, type="q8_0", padded=0, name="gate_up_181_of_60_q8"),
        # a chunk of a long prompt: the largest
        dict(kind="gate_up", tokens=2048, width=4096, hidden=14336, experts=8, top=2, type="q4_k", padded=0, name="gate_up_2048_of_8"),
        # the decode step's other half, as its files hold it
        dict(kind="down", tokens=1, width=4096, hidden=14336, experts=8, top=2, type="q6_k", padded=0, name="down_1_of_8"),
        # the eight sequences' other half
        dict(kind="down", tokens=8, width=2048, hidden=1024, experts=64, top=8, type="q4_k", padded=0, name="down_8_of_64"),
        # an odd batch with padded tokens that no expert takes
        dict(kind="down", tokens=37, width=2048, hidden=1408, experts=60, top=4, type="q8_0", padded=5, name="down_37_of_60_q8"),
        # the prompt chunk's other half
        dict(kind="down", tokens=2048, width=4096, hidden=14336, experts=8, top=2, type="q6_k", padded=0, name="down_2048_of_8"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["route", "gate_up", "gate_up", "down", "down"])
    top = rng.choice([1, 2, 2, 4, 6, 8])
    experts = _log(rng, max(4, 2 * top), 128)
    tokens = _log(rng, 1, 2048)
    if kind == "route":
        return dict(kind=kind, tokens=tokens, width=32 * _log(rng, 8, 128), experts=experts, top=top, normalize=rng.random() < 0.5)
    which = rng.choice(["q4_k", "q4_k", "q6_k", "q8_0"])
    # blocks of 256 have both sizes in whole blocks, blocks of 32 need no more than that
    unit = TYPES[which][1]
    width, hidden = unit * _log(rng, 512 // unit, 4096 // unit), unit * _log(rng, 256 // unit, 14336 // unit)
    while experts * width * hidden > 8 * 4096 * 14336:
        hidden = max(unit, hidden // 2 // unit * unit)
    while tokens * top * width * hidden > 2048 * 2 * 4096 * 14336:
        tokens = (tokens + 1) // 2
    return dict(kind=kind, tokens=tokens, width=width, hidden=hidden, experts=experts, top=top, type=which,
                padded=rng.randint(0, tokens // 4))


# ---- inputs --------------------------------------------------------------------

class Draws:
    """Seeded values on the GPU; the same calls give the same values."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda", dtype=torch.float32)

    def uniform(self, lo, hi, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda", dtype=torch.float32) * (hi - lo) + lo

    def ints(self, lo, hi, *shape, dtype=torch.uint8):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda", dtype=dtype)


def _halves(x):
    """float32 [...] -> the two bytes of its float16, [..., 2]."""
    return x.to(torch.float16).unsqueeze(-1).view(torch.uint8)


def _weights(r, which, rows, k):
    """Blocks of `rows` rows of k weights with a standard deviation of about
    0.02, as their type holds them: uint8 [rows, k / block, bytes]."""
    _, block, nbytes = TYPES[which]
    nb = k // block
    raw = r.ints(0, 256, rows, nb, nbytes)
    scale = r.uniform(0.7, 1.3, rows, nb)
    if which == "q8_0":
        raw[..., :2] = _halves(scale * (0.02 / 74))
    elif which == "q6_k":
        raw[..., 192:208] = r.ints(64, 128, rows, nb, 16)
        raw[..., 208:] = _halves(scale * (0.02 / 18.5 / 96))
    else:
        s, m = r.ints(24, 64, rows, nb, 8), r.ints(24, 64, rows, nb, 8)  # six bits each
        raw[..., 0:2] = _halves(scale * (0.02 / 4.6 / 44))
        raw[..., 2:4] = _halves(scale * (0.02 / 4.6 / 44 * 7.5))
        raw[..., 4:8] = s[..., :4] | s[..., 4:] >> 4 << 6
        raw[..., 8:12] = m[..., :4] | m[..., 4:] >> 4 << 6
        raw[..., 12:16] = s[..., 4:] & 15 | (m[..., 4:] & 15) << 4
    return raw


def _plan_shape(c):
    """int32 entries of a plan (include/mimg.h) and where the order and the
    pairs' experts begin: experts + 1 first places, then P pairs in order by
    expert, then each pair's expert, each part from a multiple of 64 on."""
    pairs = c["tokens"] * c["top"]
    order = (c["experts"] + 1 + 63) // 64 * 64
    expert = order + (pairs + 63) // 64 * 64
    return order, expert, expert + pairs


def _plan(c, ids):
    """The plan of given choices: pairs in order by expert, those of one expert
    in their own order, pairs without an expert behind all."""
    order, expert, total = _plan_shape(c)
    flat = ids.reshape(-1).long()
    plan = torch.zeros(total, device="cuda", dtype=torch.int32)
    key = torch.where(flat < 0, torch.full_like(flat, c["experts"]), flat)
    plan[1:c["experts"] + 1] = torch.bincount(key, minlength=c["experts"] + 1)[:c["experts"]].cumsum(0).int()
    plan[order:order + flat.numel()] = torch.sort(key, dim=-1, stable=True)[1].int()
    plan[expert:] = flat.int()
    return plan


def _choices(r, c):
    """Uneven choices, as trained routers make them; the padded tokens at the
    end have none."""
    gumbel = -torch.log(-torch.log(r.uniform(1e-6, 1 - 1e-6, c["tokens"], c["experts"])))
    ids = torch.topk(gumbel + 0.5 * r.normal(c["experts"]), c["top"], -1)[1].to(torch.int32)
    ids[c["tokens"] - c["padded"]:] = -1
    return ids


def _outliers(x):
    """A few channels of trained hidden states are several times the others."""
    x[..., 3::37] *= 4
    return x


def _prepare_route(c, seed):
    r = Draws(seed)
    t, n, k = c["tokens"], c["experts"], c["width"]
    # a direction that all tokens share makes some experts favourites
    x = _outliers(r.normal(t, k) + 0.3 * r.normal(k))
    router = r.normal(n, k) * (1.5 / math.sqrt(k))
    total = _plan_shape(c)[2]
    return dict(c, x=x, router=router, ids=torch.empty(t, c["top"], device="cuda", dtype=torch.int32),
                weights=torch.empty(t, c["top"], device="cuda"), plan=torch.zeros(total, device="cuda", dtype=torch.int32))


def _prepare_gate_up(c, seed):
    r = Draws(seed)
    gate, up = (_weights(r, c["type"], c["experts"] * c["hidden"], c["width"]) for _ in range(2))
    x = _outliers(r.normal(c["tokens"], c["width"]))
    ids = _choices(r, c)
    s = dict(c, gate=gate, up=up, x=x, ids=ids, plan=_plan(c, ids), h=torch.zeros(c["tokens"] * c["top"], c["hidden"], device="cuda"))
    if own:  # the handles of the layer's weights
        s.update(gate_handle=_registered(s, "gate"), up_handle=_registered(s, "up"))
    return s


def _prepare_down(c, seed):
    r = Draws(seed)
    down = _weights(r, c["type"], c["experts"] * c["width"], c["hidden"])
    pairs = c["tokens"] * c["top"]
    # what gate, up and swiglu leave: a heavy tail around zero
    h = torch.nn.functional.silu(r.normal(pairs, c["hidden"])) * r.normal(pairs, c["hidden"])
    ids = _choices(r, c)
    weights = torch.softmax(torch.sort(r.normal(c["tokens"], c["top"]), -1, descending=True)[0], -1)
    s = dict(c, down=down, h=h, ids=ids, weights=weights, plan=_plan(c, ids), y=torch.empty(c["tokens"], c["width"], device="cuda"))
    if own:
        s.update(down_handle=_registered(s, "down"))
    return s


# ---- the plain forms -------------------------------------------------------------

def _plain_weights(which, raw):
    """[..., blocks, bytes] -> float32 [..., blocks * weights of a block]."""
    if which == "q8_0":
        w = raw[..., 2:].contiguous().view(torch.int8).float() * raw[..., :2].contiguous().view(torch.float16).float()
    elif which == "q6_k":
        low, high = raw[..., :128].unflatten(-1, (2, 64)), raw[..., 128:192].unflatten(-1, (2, 32))
        low = torch.stack([low & 15, low >> 4], -2).flatten(-2).unflatten(-1, (4, 32))  # [.., half, quarter, 32]
        high = torch.stack([high & 3, high >> 2 & 3, high >> 4 & 3, high >> 6], -2)
        q = (low | high << 4).float() - 32
        scale = raw[..., 192:208].contiguous().view(torch.int8).float() * raw[..., 208:].contiguous().view(torch.float16).float()
        w = (q.flatten(-3).unflatten(-1, (16, 16)) * scale[..., None]).flatten(-2)
    else:
        d = raw[..., :4].contiguous().view(torch.float16).float()
        a, b, e = raw[..., 4:8], raw[..., 8:12], raw[..., 12:16]
        s = torch.cat([a & 63, e & 15 | a >> 6 << 4], -1).float() * d[..., :1]
        m = torch.cat([b & 63, e >> 4 | b >> 6 << 4], -1).float() * d[..., 1:]
        q = raw[..., 16:].unflatten(-1, (4, 32))
        q = torch.stack([q & 15, q >> 4], -2).flatten(-3, -2).float()  # [.., 8, 32]
        w = (q * s[..., None] - m[..., None]).flatten(-2)
    return w.flatten(-2)


def _plain_acts(x, block):
    """x in 8 bits a value and a float32 scale a block, as the values that this
    stands for; the borders between two integers are decided in 64 bits."""
    b = x.unflatten(-1, (-1, block))
    amax = b.abs().amax(-1, keepdim=True)
    q = torch.round(b.double() * 127 / torch.where(amax > 0, amax, torch.ones_like(amax)).double()).float()
    return (q * (amax.double() / 127).float()).flatten(-2)


def _plain_products(s, x, names, n):
    """x [pairs, k] times each pair's expert's matrices: a list of [pairs, n];
    zeros where a pair has no expert. The rows of an expert lie together, all
    experts' rows filled up to as many."""
    ids = s["ids"].reshape(-1).long()
    used, where = torch.unique(ids, return_inverse=True)
    count = torch.bincount(where)
    place = torch.empty_like(ids)
    by = torch.sort(where, dim=-1, stable=True)[1]
    place[by] = torch.arange(ids.numel(), device=x.device) - (count.cumsum(0) - count)[where[by]]
    padded = torch.zeros(used.numel(), int(count.max()), x.shape[1], device=x.device)
    padded[where, place] = x
    out = []
    out += [torch.matmul(padded, _plain_weights(s["type"], s[name].unflatten(0, (s["experts"], n))[used.clamp_min(0)]).transpose(1, 2))[where, place]
            * (ids >= 0)[:, None] for name in names]
    return out


def _plain_route(s):
    order, expert, _ = _plan_shape(s)
    # a choice is a step: the logits in 64 bits
    logits = torch.matmul(s["x"].double(), s["router"].double().T)
    value, ids = torch.sort(logits, dim=-1, descending=True, stable=True)
    value, ids = value[:, :s["top"]], ids[:, :s["top"]].to(torch.int32)
    total = (value if s["normalize"] else logits) - value[:, :1]
    weights = torch.exp(value - value[:, :1]) / torch.exp(total).sum(-1, keepdim=True)
    plan = _plan(s, ids)
    return dict(ids=ids, weights=weights.float(), first=plan[:s["experts"] + 1], order=plan[order:order + ids.numel()], expert=plan[expert:])


def _plain_gate_up(s):
    x = _plain_acts(s["x"], TYPES[s["type"]][1])
    gate, up = _plain_products(s, x.repeat_interleave(s["top"], 0), ("gate", "up"), s["hidden"])
    return gate / (1 + torch.exp(-gate)) * up


def _plain_down(s):
    y, = _plain_products(s, _plain_acts(s["h"], TYPES[s["type"]][1]), ("down",), s["width"])
    return (y.unflatten(0, (s["tokens"], s["top"])) * s["weights"][..., None]).sum(1)


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


def _registered(s, name):
    """All experts' matrices of one kind as one registered weight."""
    lib, raw = _library(), s[name]
    torch.cuda.synchronize()
    which, block, _ = TYPES[s["type"]]
    return lib.Weight((raw.data_ptr(), raw.numel()), which, raw.shape[0], raw.shape[1] * block, device=True)


def _workspace(s, nbytes):
    """A state's workspace, made at its first pass."""
    if "ws" not in s:
        s["ws"] = torch.empty(max(nbytes(), 256), device="cuda", dtype=torch.uint8)
    return s["ws"].data_ptr(), s["ws"].numel()


def _own_route(s):
    lib, order, expert = _library(), *_plan_shape(s)[:2]
    ws = _workspace(s, lambda: lib.experts_route_workspace_bytes(s["tokens"], s["experts"]))
    lib.experts_route_dev(s["x"].data_ptr(), s["router"].data_ptr(), s["tokens"], s["width"], s["experts"], s["top"], s["normalize"],
                          s["ids"].data_ptr(), s["weights"].data_ptr(), s["plan"].data_ptr(), s["plan"].numel() * 4, *ws,
                          torch.cuda.current_stream().cuda_stream)
    plan, pairs = s["plan"], s["ids"].numel()
    return dict(ids=s["ids"], weights=s["weights"], first=plan[:s["experts"] + 1], order=plan[order:order + pairs], expert=plan[expert:])


def _own_gate_up(s):
    lib = _library()
    ws = _workspace(s, lambda: lib.experts_swiglu_workspace_bytes(s["tokens"], s["top"], s["hidden"], s["width"]))
    lib.experts_swiglu_a8_dev(s["gate_handle"], s["up_handle"], s["experts"], s["x"].data_ptr(), s["tokens"], s["top"], s["plan"].data_ptr(),
                              s["plan"].numel() * 4, s["h"].data_ptr(), *ws, torch.cuda.current_stream().cuda_stream)
    return s["h"]


def _own_down(s):
    lib = _library()
    ws = _workspace(s, lambda: lib.experts_combine_workspace_bytes(s["tokens"], s["top"], s["width"], s["hidden"]))
    lib.experts_combine_a8_dev(s["down_handle"], s["experts"], s["h"].data_ptr(), s["weights"].data_ptr(), s["tokens"], s["top"],
                               s["plan"].data_ptr(), s["plan"].numel() * 4, s["y"].data_ptr(), *ws,
                               torch.cuda.current_stream().cuda_stream)
    return s["y"]


# ---- in 64 bits, from the definitions ------------------------------------------------

def _exact_matrix(which, raw):
    """One matrix [n, blocks, bytes] in float64, weight by weight position."""
    n, nb, _ = raw.shape
    b = raw.to(torch.int64)

    def half(at):
        return raw[..., at:at + 2].contiguous().view(torch.float16).double()

    if which == "q8_0":
        return (((b[..., 2:] + 128) % 256 - 128).double() * half(0)).reshape(n, nb * 32)
    e = torch.arange(256, device=raw.device)
    if which == "q6_k":
        part, lane = e // 32 % 4, e % 32
        low = b[..., 64 * (e // 128) + 32 * (part % 2) + lane] >> 4 * (part // 2) & 15
        high = b[..., 128 + 32 * (e // 128) + lane] >> 2 * part & 3
        scale = (b[..., 192 + e // 16] + 128) % 256 - 128
        return ((low + 16 * high - 32) * scale * half(208)).reshape(n, nb * 256)
    j = e // 32
    q = b[..., 16 + 32 * (j // 2) + e % 32] >> 4 * (j % 2) & 15
    head = b[..., 4:16]
    near, far = j % 4, j >= 4
    s = torch.where(far, (head[..., 8 + near] & 15) + 16 * (head[..., near] >> 6), head[..., near] & 63)
    m = torch.where(far, (head[..., 8 + near] >> 4) + 16 * (head[..., 4 + near] >> 6), head[..., 4 + near] & 63)
    return (q * s * half(0) - m * half(2)).reshape(n, nb * 256)


def _exact_acts(x, block):
    v = x.double().reshape(x.shape[0], -1, block)
    top = v.abs().max(-1, keepdim=True).values
    whole = torch.where(top > 0, 127 * v / top, torch.zeros_like(v)).round()
    return (whole * (top / 127).float().double()).reshape(x.shape)


def _exact_route(c, seed):
    s = _prepare_route(c, seed)
    logits = torch.cat([(part.double()[:, None, :] * s["router"].double()).sum(-1) for part in s["x"].split(16)])
    p = torch.softmax(logits, -1)
    ids = torch.argsort(logits, dim=-1, descending=True, stable=True)[:, :c["top"]]
    weights = torch.gather(p, 1, ids)
    if c["normalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    flat = ids.reshape(-1)
    first = torch.stack([(flat < e).sum() for e in range(c["experts"] + 1)])
    order = torch.cat([torch.nonzero(flat == e)[:, 0] for e in range(c["experts"])])
    return dict(ids=ids.int(), weights=weights, first=first.int(), order=order.int(), expert=flat.int())


def _by_expert(s, x, names, n):
    """Each pair's products, expert by expert."""
    flat = s["ids"].reshape(-1)
    out = [torch.zeros(flat.numel(), n, device="cuda", dtype=torch.float64) for _ in names]
    for e in range(s["experts"]):
        at = torch.nonzero(flat == e)[:, 0]
        if at.numel():
            for o, name in zip(out, names):
                o[at] = x[at] @ _exact_matrix(s["type"], s[name][e * n:(e + 1) * n]).T
    return out


def _exact_gate_up(c, seed):
    s = _prepare_gate_up(c, seed)
    x = _exact_acts(s["x"], TYPES[c["type"]][1])
    gate, up = _by_expert(s, x[torch.arange(c["tokens"] * c["top"], device="cuda") // c["top"]], ("gate", "up"), c["hidden"])
    return gate * torch.sigmoid(gate) * up


def _exact_down(c, seed):
    s = _prepare_down(c, seed)
    y, = _by_expert(s, _exact_acts(s["h"], TYPES[c["type"]][1]), ("down",), c["width"])
    return torch.einsum("tjn,tj->tn", y.reshape(c["tokens"], c["top"], -1), s["weights"].double())


# ---- the interface ---------------------------------------------------------------------

def prepare(case, seed):
    return {"route": _prepare_route, "gate_up": _prepare_gate_up, "down": _prepare_down}[case["kind"]](case, seed)


def run(state):
    if own:
        return {"route": _own_route, "gate_up": _own_gate_up, "down": _own_down}[state["kind"]](state)
    return {"route": _plain_route, "gate_up": _plain_gate_up, "down": _plain_down}[state["kind"]](state)


def exact(case, seed):
    return {"route": _exact_route, "gate_up": _exact_gate_up, "down": _exact_down}[case["kind"]](case, seed)


def work(case):
    """Inputs read and outputs written once, of the experts' weights those that
    this many tokens choose where all experts are as likely; two operations for
    each product."""
    c = case
    t, top, k = c["tokens"], c["top"], c["width"]
    if c["kind"] == "route":
        return dict(bytes=4 * (t * k + c["experts"] * k) + t * top * 16 + 4 * c["experts"], flops=2 * t * c["experts"] * k)
    t -= c["padded"]
    chosen = c["experts"] * (1 - (1 - top / c["experts"]) ** t)
    _, block, nbytes = TYPES[c["type"]]
    matrix = k * c["hidden"] // block * nbytes
    if c["kind"] == "gate_up":
        return dict(bytes=int(2 * chosen * matrix) + 4 * t * k + 4 * t * top * c["hidden"], flops=4 * t * top * k * c["hidden"])
    return dict(bytes=int(chosen * matrix) + 4 * t * top * c["hidden"] + 4 * c["tokens"] * k, flops=2 * t * top * k * c["hidden"])
