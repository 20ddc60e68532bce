"""GPU: the norms around a block against 64-bit torch.

Tolerance.  Every result is an fp32 value rounded once: half a step of its type
(2^-8 of the value for bf16, 2^-24 for fp32).  The fp32 value: the inverse root
mean square's sum has at most 16384/(T) + 16 terms after another, so its
relative error is below 128 * 2^-24 halved by the root, and with the products
after it below 2^-17 for a bf16 or fp32 row; that error is relative to the terms
that out adds up (residual and branch), and h's norm passes it on."""

import itertools

import numpy as np
import pytest
import torch

from pagedmoe_amd import _lib, kernels as K, streaming as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
F32 = 2.0 ** -17


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rms(v, w, eps, off):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * (w.double() + off)


def near(got, ref, terms, scale=1.0):
    """got is ref rounded once, its fp32 value off by F32 of terms."""
    lim = ref.abs() * HALF[got.dtype] + terms.abs() * F32 * scale + 1e-37
    err = (got.double() - ref).abs()
    assert got.shape == ref.shape and bool((err <= lim).all()), float((err / lim).max())


@pytest.mark.parametrize("stream", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("wt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,d", [(1, 1), (3, 7), (1, 8), (5, 64), (2, 312), (4, 512), (3, 520),
                                 (2, 2048), (1, 2056), (3, 4096), (2, 4104), (2, 7168), (1, 8192),
                                 (2, 8200), (1, 16384), (2, 16383), (300, 96)])
def test_norm(n, d, stream, wt):
    g = gen(n * 100000 + d)
    x = (torch.randn(n, d, device=DEV, generator=g) * 3).to(stream)
    w = torch.randn(d, device=DEV, generator=g).to(wt)
    for off in (False, True):
        h = K.block_norm(x, w, 1e-5, off)
        assert h.dtype == torch.bfloat16
        ref = rms(x.double(), w, 1e-5, float(off))
        near(h, ref, ref)


def join_ref(a):
    y = a["y"].double()
    mag = y.abs()
    if a["weights"] is not None:
        w = a["weights"].double()[..., None]
        y, mag = (y * w).sum(1), (mag * w.abs()).sum(1)
    if a["shared_y"] is not None:
        s = 1.0 if a["shared_logit"] is None else torch.sigmoid(a["shared_logit"].double())[:, None]
        y, mag = y + s * a["shared_y"].double(), mag + (s * a["shared_y"].double()).abs()
    off, eps = float(a["unit_offset"]), a["eps"]
    if a["post_weight"] is not None:
        inv = 1 / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        # the sum's own errors reach every element through the norm
        lift = ((mag * mag).mean(-1, keepdim=True) ** 0.5 * y.abs() * inv ** 2 + mag * inv)
        y = rms(y, a["post_weight"], eps, off)
        mag = lift * (a["post_weight"].double() + off).abs() + y.abs()
    if a["gate"] is not None:
        gt = a["gate"].double()
        gt = torch.sigmoid(gt) if a["gate_sigmoid"] else gt
        y, mag = y * gt, mag * gt.abs()
    r = a["residual"].double()
    out = a["residual_scale"] * r + a["branch_scale"] * y
    mag = abs(a["residual_scale"]) * r.abs() + abs(a["branch_scale"]) * mag
    if a["next_weight"] is None:
        return out, mag, None, None
    inv = 1 / torch.sqrt((out * out).mean(-1, keepdim=True) + eps)
    h = rms(out, a["next_weight"], eps, off)
    lift = ((mag * mag).mean(-1, keepdim=True) ** 0.5 * out.abs() * inv ** 2 + mag * inv)
    return out, mag, h, lift * (a["next_weight"].double() + off).abs() + h.abs()


def make(n, d, k, stream, wt, gate, post, nxt, shared, seed, gate_dtype=torch.bfloat16):
    g = gen(seed)
    rn = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    a = dict(residual=(rn(n, d) * 3).to(stream), weights=None, shared_y=None, shared_logit=None,
             post_weight=rn(d).to(wt) if post else None, next_weight=rn(d).to(wt) if nxt else None,
             gate=None, gate_sigmoid=False, residual_scale=0.9, branch_scale=-0.37, eps=1e-6,
             unit_offset=bool(seed % 2))
    a["y"] = (rn(n, k, d) if k else rn(n, d)).to(torch.bfloat16)
    if k:
        a["weights"] = rn(n, k)
    if shared:
        a["shared_y"] = rn(n, d).to(torch.bfloat16)
        a["shared_logit"] = rn(n) if shared == 2 else None
    if gate:
        a["gate"] = rn(*{"channel": (d,), "token": (n, 1), "element": (n, d)}[gate]).to(gate_dtype)
        a["gate_sigmoid"] = seed % 3 == 0
    return a


def run(a, **kw):
    b = dict(a, **kw)
    return K.block_join(b.pop("residual"), b.pop("y"), b.pop("weights"), **b)


def check(a):
    out, h = run(a)
    ref, mag, hr, hmag = join_ref(a)
    assert out.dtype == a["residual"].dtype
    near(out, ref, mag, 2)
    assert (h is None) == (hr is None)
    if h is not None:
        near(h, hr, hmag, 4)
    out2, h2 = run(a)
    assert torch.equal(out, out2) and (h is None or torch.equal(h, h2))
    return out, h


SHAPES = [(1, 1), (2, 13), (3, 64), (5, 512), (1, 2048), (4, 4096), (3, 7168), (2, 8200), (1, 16384),
          (2, 10001), (70, 312)]


@pytest.mark.parametrize("n,d", SHAPES)
@pytest.mark.parametrize("gate", [None, "channel", "token", "element"])
def test_join(n, d, gate):
    seeds = itertools.count(n * 7 + d)
    for stream, wt in itertools.product((torch.bfloat16, torch.float32), repeat=2):
        for k, post, nxt, shared in ((0, True, True, 0), (3, True, False, 0), (1, False, True, 2),
                                     (0, False, False, 1), (10, True, True, 2)):
            check(make(n, d, k, stream, wt, gate, post, nxt, shared, next(seeds),
                       gate_dtype=wt))


def test_join_combines_as_combine_does():
    """Without norm, gate and residual the result is pmoe_combine's, bit for bit."""
    a = make(9, 1024, 8, torch.bfloat16, torch.bfloat16, None, False, False, 2, 4)
    out, _ = run(a, residual_scale=0.0, branch_scale=1.0)
    assert torch.equal(out, K.combine(a["y"], a["weights"], a["shared_y"], a["shared_logit"]))


@pytest.mark.parametrize("d", [1024, 1001])
@pytest.mark.parametrize("stream", [torch.bfloat16, torch.float32])
def test_join_in_place(stream, d):
    """out may be the residual: the same bits as into an array of its own."""
    a = make(6, d, 0, stream, torch.bfloat16, "channel", True, True, 0, 8)
    out, h = run(a)
    res = a["residual"].clone()
    o2, h2 = run(a, residual=res, out=res)
    assert o2 is res and torch.equal(res, out) and torch.equal(h, h2)


def test_rows_off_16_bytes_give_the_same_rows():
    """Arrays that start off 16 bytes take the element path; its sums run in
    another order, so results agree to the bound, not in every bit."""
    a = make(4, 256, 0, torch.float32, torch.bfloat16, "element", True, True, 0, 3)
    for name in ("residual", "y", "gate", "next_weight"):
        t = a[name]
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:]
        b = dict(a, **{name: flat.view(t.shape).copy_(t)})
        assert b[name].data_ptr() % 16
        check(b)


@pytest.mark.parametrize("d", [8, 512, 520, 2048, 2056, 4096, 4104, 7168, 8192, 8200, 12288, 16384])
def test_rows_do_not_depend_on_their_number(d):
    """One row, few and many take different numbers of threads: the same bits."""
    a = make(700, d, 2, torch.bfloat16, torch.bfloat16, "element", True, True, 0, 3)
    out, h = run(a)
    nh = K.block_norm(a["residual"], a["next_weight"])
    for r0, r1 in ((0, 1), (5, 517), (699, 700)):
        part = {k: v[r0:r1].contiguous() if torch.is_tensor(v) and v.dim() >= 2 else v
                for k, v in a.items()}
        o, hh = run(part)
        assert torch.equal(out[r0:r1], o) and torch.equal(h[r0:r1], hh)
        assert torch.equal(nh[r0:r1], K.block_norm(part["residual"], a["next_weight"]))


@pytest.mark.parametrize("d", [8192, 8191])
def test_rows_past_32_bits(d):
    """More than 2^32 elements: the last rows are those of a call of their own."""
    n = 2 ** 32 // d + 100
    x = torch.empty(n, d, device=DEV, dtype=torch.bfloat16)
    x[-50:] = torch.randn(50, d, device=DEV, generator=gen(1)).to(torch.bfloat16)
    x[:-50] = 1
    w = torch.randn(d, device=DEV, generator=gen(2))
    tail = x[-50:].clone()
    assert torch.equal(K.block_norm(x, w)[-50:], K.block_norm(tail, w))
    out, h = K.block_join(x, x, gate=w, next_weight=w)
    o, hh = K.block_join(tail, tail, gate=w, next_weight=w)
    assert torch.equal(out[-50:], o) and torch.equal(h[-50:], hh)


@pytest.mark.parametrize("stream", [torch.bfloat16, torch.float32])
def test_past_the_caches(stream):
    """Results of more than 64 MiB, in place too: the rows that shorter calls give."""
    a = make(8500, 4096, 0, stream, torch.bfloat16, "element", True, True, 0, 2)
    out, h = run(a)
    nh = K.block_norm(a["residual"], a["next_weight"])
    for r0 in (0, 4000, 8400):
        part = {k: v[r0:r0 + 100].contiguous() if torch.is_tensor(v) and v.dim() == 2 else v
                for k, v in a.items()}
        o, hh = run(part)
        assert torch.equal(out[r0:r0 + 100], o) and torch.equal(h[r0:r0 + 100], hh)
        assert torch.equal(nh[r0:r0 + 100], K.block_norm(part["residual"], a["next_weight"]))
    res = a["residual"]
    o, hh = run(a, out=res)
    assert o is res and torch.equal(o, out) and torch.equal(hh, h)


def test_special_rows():
    """A zero row stays zero (eps keeps the norm finite); an infinity or NaN
    makes its own row's h NaN and no other row's."""
    w = torch.ones(512, device=DEV)
    x = torch.randn(6, 512, device=DEV, generator=gen(0))
    good = K.block_norm(x, w)
    x[1] = 0
    x[2, 5], x[3, 100] = float("inf"), float("nan")
    h = K.block_norm(x, w)
    assert (h[1] == 0).all() and torch.isnan(h[3]).all() and torch.isnan(h[2, 5])
    assert torch.equal(h[[0, 4, 5]], good[[0, 4, 5]])
    assert (K.block_norm(torch.zeros(2, 9, device=DEV), w[:9].contiguous(), 1e-6) == 0).all()
    a = make(5, 512, 2, torch.float32, torch.float32, "token", True, True, 0, 6)
    out, h = run(a)
    a["y"] = a["y"].clone()
    a["y"][3, 1, 7] = float("nan")
    o2, h2 = run(a)
    keep = [0, 1, 2, 4]
    assert torch.isnan(o2[3]).all() and torch.isnan(h2[3]).all()
    assert torch.equal(out[keep], o2[keep]) and torch.equal(h[keep], h2[keep])


def test_refusals():
    x = torch.zeros(4, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    y = torch.zeros(4, 64, device=DEV, dtype=torch.bfloat16)
    for bad in (lambda: K.block_norm(x.half(), w), lambda: K.block_norm(x, w.half()),
                lambda: K.block_norm(x, w[:32].contiguous()), lambda: K.block_norm(x[:, ::2], w),
                lambda: K.block_norm(x[0], w), lambda: K.block_norm(x, w, -1.0),
                lambda: K.block_norm(torch.zeros(1, 16392, device=DEV), torch.zeros(16392, device=DEV)),
                lambda: K.block_join(x, y.float()), lambda: K.block_join(x, y[:3].contiguous()),
                lambda: K.block_join(x, y.reshape(4, 1, 64)),
                lambda: K.block_join(x, y, torch.ones(4, 1, device=DEV)),
                lambda: K.block_join(x, y, gate=torch.ones(4, device=DEV)),
                lambda: K.block_join(x, y, gate=torch.ones(4, 2, device=DEV)),
                lambda: K.block_join(x, y, post_weight=w, next_weight=w.to(torch.bfloat16)),
                lambda: K.block_join(x, y, shared_logit=torch.zeros(4, device=DEV)),
                lambda: K.block_join(x, y, out=torch.zeros(4, 64, device=DEV, dtype=torch.bfloat16)),
                lambda: K.block_join(x, y, out=torch.zeros(3, 64, device=DEV)),
                lambda: K.block_norm(x.cpu(), w), lambda: K.block_join(x, y, gate=w.cpu())):
        with pytest.raises((TypeError, ValueError, _lib.PmoeError)):
            bad()
    e = x[:0]
    assert K.block_norm(e, w).shape == (0, 64)
    out, h = K.block_join(e, y[:0], next_weight=w)
    assert out.shape == h.shape == (0, 64)


def test_stream_and_capture():
    a = make(33, 2048, 4, torch.bfloat16, torch.bfloat16, "element", True, True, 1, 5)
    out, h = run(a)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        o2, h2 = run(a)
        n2 = K.block_norm(a["residual"], a["next_weight"])
    st.synchronize()
    assert torch.equal(out, o2) and torch.equal(h, h2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o3, h3 = run(a)
        n3 = K.block_norm(a["residual"], a["next_weight"])
    for i in range(3):
        a["residual"].add_(1)
        graph.replay()
        torch.cuda.synchronize()
        out, h = run(a)
        assert torch.equal(out, o3) and torch.equal(h, h3)
        assert torch.equal(n3, K.block_norm(a["residual"], a["next_weight"]))
    assert not torch.equal(n2, n3)


@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("paged", [False, True])
def test_layers(group, paged):
    """Two MoE layers one after the other, the first's join making the second's
    input: as norm, block, combine and join one by one, for a prompt in several
    fetch groups and single tokens."""
    hidden, inter, experts, k = 512, 128, 16, 4
    g = gen(2)
    rn = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    layers = torch.nn.ModuleList()
    for li in range(2):
        glu = S.QuantizedSwitchGLU(hidden, inter, experts, 4, group, n_shared=1)
        for e in range(experts + 1):
            glu.quantize_expert(e, rn(inter, hidden) * 0.05, rn(inter, hidden) * 0.05,
                                rn(hidden, inter) * 0.05)
        blk = S.SoftmaxMoEBlock(rn(experts, hidden) * 0.1, glu, k,
                                shared_expert_gate=rn(1, hidden) * 0.1)
        layers.append(S.MoELayer(blk, 0.1 * rn(hidden), 0.1 * rn(hidden) if li else None,
                                 rn(hidden), gate_sigmoid=True, residual_scale=0.9,
                                 branch_scale=0.3, unit_offset=True))
    if paged:
        cache = S.build_cache_for(layers, slots=12)
        S.patch_model(layers, cache, predict_mode="off")
        assert layers[0].block.switch_mlp.cache is cache
    for n in (1, 3, 100):
        x = rn(n, hidden)
        h1 = layers[1].pre_weight
        a, ha = layers[0](x, next_weight=h1)
        b = layers[1](a, h=ha)
        # one by one
        r = x.double()
        for li, lay in enumerate(layers):
            xin = r.float()
            hn = K.block_norm(xin, lay.pre_weight, lay.eps, True)
            y = lay.block(hn.reshape(1, n, hidden)).reshape(n, hidden)
            out, _ = K.block_join(xin, y, post_weight=lay.post_weight, gate=lay.gate,
                                  gate_sigmoid=True, residual_scale=0.9, branch_scale=0.3,
                                  unit_offset=True)
            r = out.double()
        # h and the combined block output are rounded to bf16 on one side only
        assert (b.double() - r).norm() <= 2.0 ** -7 * r.norm()
    y = layers[0].block(x.to(torch.bfloat16).reshape(2, 50, hidden))
    assert y.shape == (2, 50, hidden)


def test_layer_gates_beside_leading_dims():
    """A gate given in x's own leading dims is the one of the flat rows."""
    hidden, inter, experts = 256, 128, 8
    g = gen(4)
    rn = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    glu = S.QuantizedSwitchGLU(hidden, inter, experts, 4, 32)
    for e in range(experts):
        glu.quantize_expert(e, rn(inter, hidden) * 0.05, rn(inter, hidden) * 0.05,
                            rn(hidden, inter) * 0.05)
    layer = S.MoELayer(S.SoftmaxMoEBlock(rn(experts, hidden) * 0.1, glu, 2), torch.ones(hidden, device=DEV),
                       gate_sigmoid=True)
    x = rn(2, 5, hidden)
    for gate in (rn(2, 5, 1), rn(2, 5, hidden)):
        out = layer(x, gate=gate)
        flat = layer(x.reshape(10, hidden), gate=gate.reshape(10, -1))
        assert out.shape == x.shape and torch.equal(out.reshape(10, hidden), flat)
