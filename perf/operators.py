"""Microscaled 4-bit experts and the norms around a MoE block, as measurable cases.

Three operators and what a user's program has of each:

  format   weights into the microscaled 4-bit format and back: groups of 32
           values along a row share one power of two (uint8, biased by 127),
           each value is a 4-bit float of 1 sign, 2 exponent and 1 mantissa bit
  experts  the routed SwiGLU experts over such weights, at the expert seam
           (per-slot outputs [n, k, hidden]) or combined with the routing
           weights and a shared expert ([n, hidden])
  norm     the RMS norm of a residual stream before a block; and after it, in
           one pass: the combine of its slots, the norm of its output, its
           gate, the scaled residual add and the next block's norm

Shapes are the ones that the benchmark and the tests use:

  tiny  hidden 1024, inter  512,  32 experts, top-4
  q235  hidden 4096, inter 1536, 128 experts, top-8  (Qwen3-235B-shaped)
  next  hidden 2048, inter  512, 512 experts, top-10, a sigmoid-gated shared
        expert  (Qwen3-Next-shaped)
  dsv3  hidden 7168, inter 2048, 384 experts, top-8, a shared expert
        (DeepSeek-V3-shaped)

The experts of a layer lie in one buffer, an expert a slot: gate, up and down
projection, of each the packed words and then the scales, every part on 256
bytes.
"""

from __future__ import annotations

import math

import torch

own = False

SHAPES = {
    "tiny": dict(hidden=1024, inter=512, experts=32, k=4, shared=0, shared_gate=0),
    "q235": dict(hidden=4096, inter=1536, experts=128, k=8, shared=0, shared_gate=0),
    "next": dict(hidden=2048, inter=512, experts=512, k=10, shared=1, shared_gate=1),
    "dsv3": dict(hidden=7168, inter=2048, experts=384, k=8, shared=1, shared_gate=0),
}
GROUP = 32
STD = 0.02
EPS = 1e-6
# what the 16 codes stand for
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------- the cases

def listed() -> list:
    return [
        # one small ragged matrix, as a test or an adapter's weight: latency
        {"name": "format_37x96_bf16", "kind": "format", "rows": 37, "cols": 96, "dtype": "bf16"},
        # making a checkpoint: a stack of gate projections
        {"name": "format_24576x4096_fp32", "kind": "format", "rows": 24576, "cols": 4096,
         "dtype": "fp32"},
        # one token of a small model: nothing but latency and launches
        _experts("seam_tiny_1", "tiny", 1, "seam"),
        # interactive decode of one sequence
        _experts("experts_q235_1", "q235", 1, "mixture"),
        # three sequences of a large model, a shared expert
        _experts("experts_dsv3_3", "dsv3", 3, "mixture"),
        # a batch of an odd size over many small experts, a gated shared one
        _experts("experts_next_29", "next", 29, "mixture"),
        # a fetch group of a paged prompt: the seam with the slots of experts
        # that are in other groups dropped
        _experts("seam_q235_100_part", "q235", 100, "seam", part=True),
        # the largest chunk of a prompt under a trained router's uneven loads
        _experts("experts_q235_16384", "q235", 16384, "mixture", skew=True),
        # before a block: one token's residual stream
        {"name": "norm_1x4096", "kind": "norm", "n": 1, "hidden": 4096, "stream": "bf16"},
        # after a block of one short decode batch, everything fused, and the
        # next block's norm
        {"name": "join_5x7168", "kind": "join", "n": 5, "hidden": 7168, "k": 1,
         "stream": "fp32", "gate": "channel", "post": True, "next": True},
        # a paged prompt's per-slot outputs combined and joined
        {"name": "join_1000x2048_k10", "kind": "join", "n": 1000, "hidden": 2048, "k": 10,
         "stream": "bf16", "gate": "token", "post": True, "next": True},
        # a long prompt's stream
        {"name": "join_16384x4096", "kind": "join", "n": 16384, "hidden": 4096, "k": 1,
         "stream": "bf16", "gate": "element", "post": True, "next": True},
    ]


def _experts(name, shape, n, form, skew=False, part=False):
    return {"name": name, "kind": "experts", "shape": shape, "n": n, "form": form, "skew": skew,
            "part": part}


# most tokens of a drawn call: no case costs more than the 16384-token one
MOST_TOKENS = {"tiny": 16384, "q235": 8192, "next": 4096, "dsv3": 8}


def draw(rng) -> dict:
    kind = rng.choices(["format", "experts", "norm", "join"], [2, 6, 1, 3])[0]
    if kind == "format":
        return {"kind": kind, "rows": _log_int(rng, 1, 24576), "cols": 32 * _log_int(rng, 1, 224),
                "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if kind == "experts":
        shape = rng.choices(["tiny", "q235", "next", "dsv3"], [2, 3, 2, 1])[0]
        n = _log_int(rng, 1, MOST_TOKENS[shape])
        form = rng.choice(["seam", "mixture"])
        return {"kind": kind, "shape": shape, "n": min(n, 2048) if form == "seam" else n,
                "form": form, "skew": n > 64 and rng.random() < 0.5,
                "part": form == "seam" and n >= 8 and rng.random() < 0.3}
    hidden = rng.choice([1024, 2048, 4096, 7168, 8 * _log_int(rng, 8, 1024)])
    n = _log_int(rng, 1, 16384)
    if kind == "norm":
        return {"kind": kind, "n": n, "hidden": hidden, "stream": rng.choice(["bf16", "fp32"])}
    return {"kind": kind, "n": n, "hidden": hidden, "k": rng.choice([1, 1, 4, 8, 10]) if n <= 2048 else 1,
            "stream": rng.choice(["bf16", "fp32"]),
            "gate": rng.choice(["none", "channel", "token", "element"]),
            "post": rng.random() < 0.8, "next": rng.random() < 0.8}


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# ---------------------------------------------------------------- inputs

def _gen(seed: int, what: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + what) % (1 << 62))


def _normal(shape, seed: int, what: int) -> torch.Tensor:
    return torch.randn(shape, device="cuda", generator=_gen(seed, what))


def _slot(hidden: int, inter: int):
    """Byte offsets of an expert's parts in its slot, [gate, up, down] of
    (words, scales), and the slot's size."""
    offs, at = [], 0
    for _ in range(3):
        pair = []
        for size in (hidden * inter // 2, hidden * inter // GROUP):
            pair.append(at)
            at += -(-size // 256) * 256
        offs.append(tuple(pair))
    return offs, at


def _views(slab: torch.Tensor, hidden: int, inter: int):
    """[(words int32 [slots, rows, cols / 8], scales uint8 [slots, rows, cols / 32])]
    of the gate, up and down projections in a slab."""
    offs, size = _slot(hidden, inter)
    slots = slab.numel() // size
    out = []
    for (w, s), (rows, cols) in zip(offs, ((inter, hidden), (inter, hidden), (hidden, inter))):
        out.append((slab.view(torch.int32).as_strided((slots, rows, cols // 8), (size // 4, cols // 8, 1), w // 4),
                    slab.as_strided((slots, rows, cols // GROUP), (size, cols // GROUP, 1), s)))
    return out


def _slab(sh: dict, seed: int) -> torch.Tensor:
    """Experts as a quantizer leaves bell-shaped weights of STD: the largest
    of a group takes the upper two codes and the others spread nearly evenly
    over the sixteen; scales of 2^-8 to 2^-6."""
    size = _slot(sh["hidden"], sh["inter"])[1]
    slots = sh["experts"] + sh["shared"]
    gen = _gen(seed, 1)
    slab = torch.empty(slots * size, dtype=torch.uint8, device="cuda")
    slab.view(torch.int64).random_(generator=gen)
    for _, s in _views(slab, sh["hidden"], sh["inter"]):
        s.copy_(torch.randint(119, 122, s.shape, dtype=torch.uint8, device="cuda", generator=gen))
    return slab


def _hidden(n: int, d: int, seed: int) -> torch.Tensor:
    """Normalised hidden states: a few channels are much larger, as in
    trained models."""
    x = _normal((n, d), seed, 2)
    big = torch.rand(d, device="cuda", generator=_gen(seed, 3)) < 1 / 256
    return torch.where(big, 20 * x, x).to(torch.bfloat16)


def _routing(case: dict, seed: int):
    """Distinct expert ids per token, unevenly popular, and weights."""
    sh = SHAPES[case["shape"]]
    gen = _gen(seed, 5)
    pop = torch.randn(sh["experts"], device="cuda", generator=gen) * (1.0 if case["skew"] else 0.3)
    u = torch.rand((case["n"], sh["experts"]), device="cuda", generator=gen).clamp_(1e-9, 1 - 1e-7)
    z, inds = torch.topk(pop - torch.log(-torch.log(u)), sh["k"], dim=-1)
    inds = inds.to(torch.int32)
    if case["part"]:
        inds = torch.where(inds % 3 == 0, inds, torch.full_like(inds, -1))
    return inds, torch.softmax(z, -1)


def prepare(case: dict, seed: int) -> dict:
    kind = case["kind"]
    if kind == "format":
        w = _normal((case["rows"], case["cols"]), seed, 1) * STD
        return {"case": case, "w": w.to(DTYPES[case["dtype"]])}
    if kind == "experts":
        sh = SHAPES[case["shape"]]
        inds, wts = _routing(case, seed)
        st = {"case": case, "slab": _slab(sh, seed), "x": _hidden(case["n"], sh["hidden"], seed),
              "inds": inds, "weights": wts,
              "table": torch.arange(sh["experts"], dtype=torch.int32, device="cuda"),
              "shared_gate": None,
              # most rows that one expert has
              "most": int(torch.bincount(inds[inds >= 0], minlength=1).max())}
        if sh["shared_gate"]:
            st["shared_gate"] = (_normal((1, sh["hidden"]), seed, 6) * STD).to(torch.bfloat16)
        return st
    n, d = case["n"], case["hidden"]
    st = {"case": case, "residual": (_normal((n, d), seed, 1) * 3.0).to(DTYPES[case["stream"]]),
          "next": (1 + 0.1 * _normal((d,), seed, 2)).to(torch.bfloat16)}
    if kind == "norm":
        return st
    st["post"] = (1 + 0.1 * _normal((d,), seed, 3)).to(torch.bfloat16) if case["post"] else None
    if not case["next"]:
        st["next"] = None
    k = case["k"]
    st["y"] = (_normal((n, k, d) if k > 1 else (n, d), seed, 4) * 0.5).to(torch.bfloat16)
    st["weights"] = torch.softmax(_normal((n, k), seed, 5), -1) if k > 1 else None
    shape = {"none": None, "channel": (d,), "token": (n, 1), "element": (n, d)}[case["gate"]]
    st["gate"] = (0.5 * _normal(shape, seed, 6)).to(torch.bfloat16) if shape else None
    return st


# ---------------------------------------------------------------- one pass

RESIDUAL_SCALE, BRANCH_SCALE = 0.9, 0.22  # of a depth-scaled model
_GEOMS: dict = {}


def run(state: dict):
    case = state["case"]
    kind = case["kind"]
    if own:
        return _OWN[kind](state)
    return _PLAIN[kind](state)


def _own_format(st):
    from pagedmoe_amd import kernels as K
    q, s = K.mx4_quantize(st["w"])
    return K.mx4_dequant(q, s, st["w"].dtype)


def _own_experts(st):
    from pagedmoe_amd import _lib
    from pagedmoe_amd import kernels as K
    case, sh = st["case"], SHAPES[st["case"]["shape"]]
    g = _GEOMS.get(case["shape"])
    if g is None:
        g = _GEOMS[case["shape"]] = _lib.geom(sh["hidden"], sh["inter"], 4, GROUP)
    if case["form"] == "seam":
        return K.switch_glu(g, st["slab"], st["table"], sh["experts"], st["x"], st["inds"])
    return K.moe_experts(g, st["slab"], st["table"], sh["experts"], st["x"], st["inds"], st["weights"],
                         sh["experts"] if sh["shared"] else -1, st["shared_gate"])


def _own_norm(st):
    from pagedmoe_amd import kernels as K
    return K.block_norm(st["residual"], st["next"], EPS)


def _own_join(st):
    from pagedmoe_amd import kernels as K
    out, h = K.block_join(st["residual"], st["y"], st["weights"], post_weight=st["post"],
                          gate=st["gate"], residual_scale=RESIDUAL_SCALE,
                          branch_scale=BRANCH_SCALE, next_weight=st["next"], eps=EPS)
    return [out] if h is None else [out, h]


_OWN = {"format": _own_format, "experts": _own_experts, "norm": _own_norm, "join": _own_join}


# plain forms ------------------------------------------------------

_LUTS: dict = {}


def _lut(what: str) -> torch.Tensor:
    """The 16 code values, or the 256 scales, as an fp32 table."""
    if what not in _LUTS:
        vals = E2M1 if what == "codes" else [2.0 ** (i - 127) for i in range(255)] + [math.nan]
        _LUTS[what] = torch.tensor(vals, dtype=torch.float32, device="cuda")
    return _LUTS[what]


def _plain_values(words: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """fp32 [..., cols] of words [..., cols / 8] and scales [..., cols / 32]."""
    shifts = torch.arange(0, 32, 4, dtype=torch.int32, device=words.device)
    codes = torch.bitwise_and(words[..., None] >> shifts, 15)
    v = _lut("codes")[codes].reshape(*scales.shape, GROUP)
    return (v * _lut("scales")[scales.int()][..., None]).reshape(*words.shape[:-1], -1)


def _plain_format(st):
    w = st["w"].float().reshape(-1, GROUP)
    # power of two: of the largest magnitude, less the 2 that the largest code has
    e = (torch.frexp(w.abs().amax(-1)).exponent - 1 - 2).clamp(-127, 127)
    scale = _lut("scales")[e + 127][:, None]
    a = (w / scale).abs()
    # the nearest magnitude; a tie goes to the even code
    i = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    v = torch.where(w < 0, -_lut("codes")[i], _lut("codes")[i]) * scale
    return v.reshape(st["w"].shape).to(st["w"].dtype)


def _plain_glu(x, gate, up, down):
    """x [b, rows, hidden] through b experts' weights, fp32."""
    g = torch.bmm(x, gate.transpose(1, 2).contiguous())
    u = torch.bmm(x, up.transpose(1, 2).contiguous())
    return torch.bmm(g * torch.sigmoid(g) * u, down.transpose(1, 2).contiguous())


def _plain_experts(st):
    case, sh = st["case"], SHAPES[st["case"]["shape"]]
    n, k, d, e = case["n"], sh["k"], sh["hidden"], sh["experts"]
    x = st["x"].float()
    parts = _views(st["slab"], d, sh["inter"])
    ids = st["inds"].flatten().long()
    held = ids >= 0
    if n * k <= e:  # each row with its own expert's weights
        slots = st["table"][ids.clamp_min(0)].long()
        rows = x.repeat_interleave(k, 0)[:, None]
        y = _plain_glu(rows, *(_plain_values(w[slots], s[slots]) for w, s in parts))[:, 0]
    else:           # every expert's rows, as many as the fullest has
        key = torch.where(held, ids, torch.full_like(ids, e))
        order = torch.argsort(key, stable=True)
        start = torch.searchsorted(key[order], torch.arange(e + 1, device=key.device))
        place = torch.empty_like(key)
        place[order] = torch.arange(n * k, device=key.device) - start[key[order]]
        place = torch.where(held, place, torch.zeros_like(place))
        xs = torch.zeros((e + 1, st["most"], d), device=x.device)
        xs[key, place] = x.repeat_interleave(k, 0)
        slots = st["table"].long()
        y = _plain_glu(xs[:e], *(_plain_values(w[slots], s[slots]) for w, s in parts))
        y = y[key.clamp_max(e - 1), place]
    y = torch.where(held[:, None], y, torch.zeros_like(y)).reshape(n, k, d)
    if case["form"] == "seam":
        return y.to(torch.bfloat16)
    out = (y * st["weights"][..., None]).sum(1)
    if sh["shared"]:
        ys = _plain_glu(x[None], *(_plain_values(w[e:], s[e:]) for w, s in parts))[0]
        if st["shared_gate"] is not None:
            ys = ys * torch.sigmoid((x * st["shared_gate"].float()).sum(-1, keepdim=True))
        out = out + ys
    return out.to(torch.bfloat16)


def _plain_rms(v, weight):
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * weight.float()


def _plain_norm(st):
    return _plain_rms(st["residual"].float(), st["next"]).to(torch.bfloat16)


def _plain_join(st):
    y = st["y"].float()
    if st["weights"] is not None:
        y = (y * st["weights"][..., None]).sum(1)
    if st["post"] is not None:
        y = _plain_rms(y, st["post"])
    if st["gate"] is not None:
        y = y * st["gate"].float()
    out = RESIDUAL_SCALE * st["residual"].float() + BRANCH_SCALE * y
    if st["next"] is None:
        return [out.to(st["residual"].dtype)]
    return [out.to(st["residual"].dtype), _plain_rms(out, st["next"]).to(torch.bfloat16)]


_PLAIN = {"format": _plain_format, "experts": _plain_experts, "norm": _plain_norm,
          "join": _plain_join}


# ---------------------------------------------------------------- what it cannot do without

def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "format":  # values in, words and scales out; those in, values out
        vals = case["rows"] * case["cols"]
        item = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": 2 * item * vals + vals + vals // 16, "flops": 6 * vals}
    if kind == "experts":
        sh = SHAPES[case["shape"]]
        d, i, e, k, n = sh["hidden"], sh["inter"], sh["experts"], sh["k"], case["n"]
        share = 1 / 3 if case["part"] else 1.0
        mixture = case["form"] == "mixture"
        shared = sh["shared"] if mixture else 0
        seen = share * e * (1.0 - (1.0 - k / e) ** n) + shared
        rows = n * (k * share + shared)
        io = 2 * n * d + 4 * n * k + (2 * n * d + 4 * n * k if mixture else 2 * n * k * d)
        return {"bytes": int(seen * (3 * d * i // 2 + 3 * d * i // GROUP) + io),
                "flops": int(6.0 * d * i * rows)}
    n, d = case["n"], case["hidden"]
    item = 4 if case["stream"] == "fp32" else 2
    if kind == "norm":
        return {"bytes": n * d * (item + 2) + 2 * d, "flops": 4 * n * d}
    k = case["k"]
    gate = {"none": 0, "channel": d, "token": n, "element": n * d}[case["gate"]]
    size = n * d * (2 * item + 2 * k) + (4 * n * k if k > 1 else 0) + 2 * gate
    if case["next"]:
        size += 2 * n * d + 2 * d
    if case["post"]:
        size += 2 * d
    return {"bytes": size, "flops": n * d * (2 * k + 10)}


# ---------------------------------------------------------------- 64 bits

def exact(case: dict, seed: int):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "format":
        w = st["w"].double().reshape(-1, GROUP)
        top = w.abs().amax(-1, keepdim=True)
        e = torch.floor(torch.log2(top))
        # log2 may round up to a whole number just below a power of two, or down
        e = torch.where(torch.exp2(e) > top, e - 1, e)
        e = torch.where(torch.exp2(e + 1) <= top, e + 1, e)
        unit = torch.exp2((e - 2).clamp(-127, 127))
        a = (w / unit).abs().clamp_max(6.0)
        # steps of 1/2 up to 2, 1 up to 4 and 2 beyond; round() takes ties to even
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
        return (torch.sign(w) * torch.round(a / step) * step * unit).reshape(st["w"].shape)
    if kind == "experts":
        return _exact_experts(case, st)
    r = st["residual"].double()

    def rms(v, weight):
        return v / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS) * weight.double()

    if kind == "norm":
        return rms(r, st["next"])
    y = st["y"].double()
    if st["weights"] is not None:
        y = torch.matmul(st["weights"].double()[:, None], y)[:, 0]
    if st["post"] is not None:
        y = rms(y, st["post"])
    if st["gate"] is not None:
        y = y * st["gate"].double()
    out = RESIDUAL_SCALE * r + BRANCH_SCALE * y
    return [out] if st["next"] is None else [out, rms(out, st["next"])]


def _exact_experts(case: dict, st: dict):
    sh = SHAPES[case["shape"]]
    n, k, d = case["n"], sh["k"], sh["hidden"]
    parts = _views(st["slab"], d, sh["inter"])
    x = st["x"].double()
    values = torch.tensor(E2M1, dtype=torch.float64, device=x.device)

    def weight(proj, slot):
        words, scales = parts[proj][0][slot].contiguous(), parts[proj][1][slot]
        b = words.view(torch.uint8)
        v = torch.stack((values[(b & 15).int()], values[(b >> 4).int()]), -1)
        unit = torch.exp2(scales.double() - 127)
        return (v.reshape(*scales.shape, GROUP) * unit[..., None]).reshape(scales.shape[0], -1)

    def ffn(rows, slot):
        g = rows @ weight(0, slot).T
        return (g / (1 + torch.exp(-g)) * (rows @ weight(1, slot).T)) @ weight(2, slot).T

    mixture = case["form"] == "mixture"
    out = torch.zeros((n, d) if mixture else (n, k, d), dtype=torch.float64, device=x.device)
    inds = st["inds"]
    for e in torch.unique(inds).tolist():
        if e < 0:
            continue
        tok, col = (inds == e).nonzero(as_tuple=True)
        y = ffn(x[tok], int(st["table"][e]))
        if mixture:
            out.index_add_(0, tok, y * st["weights"].double()[tok, col][:, None])
        else:
            out[tok, col] = y
    if mixture and sh["shared"]:
        y = ffn(x, sh["experts"])
        if st["shared_gate"] is not None:
            y = y * torch.sigmoid(x @ st["shared_gate"].double()[0])[:, None]
        out += y
    return out
