"""GPU: the microscaled 4-bit format and its experts against 64-bit numpy.

The format is exact.  An expert output may differ from the 64-bit one by the
bound that mx_oracle.ffn derives for the fp32 value and by one rounding to
bf16 (half a step, 2^-8 of the value); over a whole output the roundings (x and h
pieces, each no worse than a rounding to bf16, and the output's own) are
independent, so the relative L2 error stays below sqrt(3) 2^-8 < 7e-3."""

import numpy as np
import pytest
import torch

from pagedmoe_amd import _lib, kernels as K, streaming as S
from pagedmoe_amd.slab import SlabStore, component_specs
from tests import mx_oracle as M

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# ---------------------------------------------------------------- format

def check_format(w, dtype):
    t = torch.from_numpy(w).to(DEV).to(dtype)
    ref_c, ref_s = M.quantize(t.double().cpu().numpy())
    q, s = K.mx4_quantize(t)
    assert np.array_equal(s.cpu().numpy(), ref_s)
    assert np.array_equal(q.cpu().numpy().view(np.uint32), M.pack(ref_c))
    for out in (torch.float32, torch.bfloat16, torch.float16):
        got = K.mx4_dequant(q, s, out)
        want = torch.from_numpy(M.dequant(ref_c, ref_s)).to(torch.float32).to(out)
        assert got.dtype == out and torch.equal(got.cpu().nan_to_num(nan=1e4), want.nan_to_num(nan=1e4))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 64), (3, 96), (65, 32), (7, 2080), (130, 1536)])
def test_format(rows, cols, dtype):
    rng = np.random.default_rng(rows * 1000 + cols)
    w = rng.standard_normal((rows, cols)).astype(np.float32)
    w *= np.exp2(rng.integers(-20, 12, (rows, 1))).astype(np.float32)
    check_format(w, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_format_edges(dtype):
    """Ties of every step in both signs, zeros and negative zeros, the ends of
    the exponent range, denormals, infinities and NaN in a group."""
    w = np.zeros((14, 64), np.float32)
    mids = ((M.E2M1[1:] + M.E2M1[:-1]) / 2).astype(np.float32)
    for r, unit in enumerate((1.0, 2.0 ** -30, 2.0 ** 100, 2.0 ** -126)):
        w[r, :7], w[r, 8:15], w[r, 16] = mids * unit, -mids * unit, 7.5 * unit
        w[r, 32:40] = M.E2M1 * unit
    w[4] = -0.0
    w[5, 3] = 2.0 ** -133  # a bf16 denormal
    w[6, :4] = [3.38e38, -3.38e38, 1e38, 1.0]
    w[7, 40] = np.inf
    w[8, 1] = -np.inf
    w[9, 63] = np.nan
    w[10, :] = 2.0 ** -128
    w[11, 0], w[11, 1] = 2.0 ** -126, 2.0 ** -127
    w[12, 0] = 6.0
    w[13, 0], w[13, 1] = 4.0, 1e-30
    check_format(w, dtype)


def test_format_unaligned_and_into_views():
    """Arrays that start off 16 bytes; a slab's components as the outputs."""
    rng = np.random.default_rng(1)
    flat = torch.from_numpy(rng.standard_normal(5 * 96 + 1).astype(np.float32)).to(DEV)
    w = flat[1:].reshape(5, 96)
    q, s = K.mx4_quantize(w)
    q2, s2 = K.mx4_quantize(w.clone())
    assert torch.equal(q, q2) and torch.equal(s, s2)
    half = flat.to(torch.bfloat16)[1:].reshape(5, 96)
    assert torch.equal(K.mx4_quantize(half)[0], K.mx4_quantize(half.clone())[0])
    slab = SlabStore(_lib.geom(96, 64, 4, 32), 3)
    slab.quantize_into(1, "down_proj", torch.ones(96, 64, device=DEV))
    assert (K.mx4_dequant(slab.expert("down_proj.weight", 1), slab.expert("down_proj.scales", 1))
            == 1).all()
    touched = slab.buf.reshape(3, -1).any(1).tolist()
    assert touched == [False, True, False]


def test_format_refusals():
    w = torch.zeros(4, 64, device=DEV)
    with pytest.raises(ValueError):
        K.mx4_quantize(w[:, :48].contiguous())
    with pytest.raises(ValueError):
        K.mx4_quantize(w[:, ::2])
    with pytest.raises(ValueError):
        K.mx4_quantize(w.reshape(-1))
    q, s = K.mx4_quantize(w)
    with pytest.raises(ValueError):
        K.mx4_dequant(q, s[:, :1].contiguous())
    with pytest.raises(TypeError):
        K.mx4_dequant(q, s, torch.float64)
    with pytest.raises(ValueError):
        K.mx4_quantize(w, out=(q, s[:3].contiguous()))
    q0, s0 = K.mx4_quantize(w[:0])
    assert q0.shape == (0, 8) and K.mx4_dequant(q0, s0).shape == (0, 64)


def test_format_long_arrays():
    """More groups than one wave of blocks and an odd count of them."""
    g = torch.Generator(device=DEV).manual_seed(0)
    w = torch.randn(4099, 4000 // 32 * 32, device=DEV, generator=g)
    q, s = K.mx4_quantize(w)
    back = K.mx4_dequant(q, s, torch.float32)
    rows = [0, 1, 2048, 4098]
    c, sc = M.quantize(w[rows].double().cpu().numpy())
    assert np.array_equal(back[rows].double().cpu().numpy(), M.dequant(c, sc))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_format_past_the_caches(dtype):
    """Results of more than 64 MiB: the same values as in parts below that."""
    g = torch.Generator(device=DEV).manual_seed(1)
    w = torch.randn(4100, 8192, device=DEV, generator=g).to(dtype)
    q, s = K.mx4_quantize(w)
    whole = K.mx4_dequant(q, s, dtype)
    for a in range(0, 4100, 1025):
        part = K.mx4_dequant(q[a:a + 1025].contiguous(), s[a:a + 1025].contiguous(), dtype)
        assert torch.equal(whole[a:a + 1025], part)


# ---------------------------------------------------------------- experts

class Layer:
    """Random experts in a slab, and their 64-bit values."""

    def __init__(self, hidden, inter, experts, shared=0, seed=0, slots=None, perm=False, scales=(118, 122)):
        rng = np.random.default_rng(seed)
        self.g = _lib.geom(hidden, inter, 4, 32)
        self.e, self.shared = experts, shared
        total = experts + shared
        self.slab = SlabStore(self.g, total if slots is None else slots)
        ids = rng.permutation(total) if perm else np.arange(total)
        self.slot = ids
        self.w = []
        for e in range(total):
            mats, comps = [], {}
            for proj, rows, cols in (("gate_proj", inter, hidden), ("up_proj", inter, hidden),
                                     ("down_proj", hidden, inter)):
                codes = rng.integers(0, 16, (rows, cols)).astype(np.uint8)
                sc = rng.integers(*scales, (rows, cols // 32)).astype(np.uint8)
                comps[proj + ".weight"], comps[proj + ".scales"] = M.pack(codes), sc
                mats.append((codes, sc))
            self.slab.write_expert(int(ids[e]), comps)
            self.w.append(mats)
        self.table = torch.from_numpy(ids[:experts].astype(np.int32)).to(DEV)
        self.shared_slot = int(ids[experts]) if shared else -1

    def ffn(self, e, x):
        return M.ffn(x, *(M.dequant(c, s) for c, s in self.w[e]))

    def seam(self, x, inds):
        n, k = inds.shape
        d = x.shape[1]
        y, b = np.zeros((n, k, d)), np.zeros((n, k, d))
        for e in np.unique(inds):
            if not 0 <= e < self.e:
                continue
            tok, col = np.nonzero(inds == e)
            y[tok, col], b[tok, col] = self.ffn(e, x[tok])
        return y, b


def bf16(a):
    return torch.from_numpy(np.asarray(a, np.float32)).to(torch.bfloat16).to(DEV)


def check(got, ref, bound, what=""):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all(), what
    lim = bound * (1 + 2.0 ** -8) + np.abs(ref) * 2.0 ** -8 + 1e-37
    bad = np.abs(got - ref) > lim
    assert not bad.any(), (what, int(bad.sum()), float((np.abs(got - ref) / lim).max()))
    norm = np.linalg.norm(ref)
    assert np.linalg.norm(got - ref) <= 7e-3 * norm, (what, np.linalg.norm(got - ref) / max(norm, 1e-300))


def tokens(rng, n, hidden, big=True):
    x = rng.standard_normal((n, hidden))
    if big:  # a few channels far above the others
        x[:, rng.random(hidden) < 0.02] *= 30
    return bf16(x)


@pytest.mark.parametrize("hidden,inter,experts,n,k", [
    (32, 32, 2, 1, 1), (32, 32, 4, 5, 2), (96, 160, 5, 7, 3), (160, 32, 3, 33, 2),
    (512, 512, 8, 3, 4), (544, 96, 8, 17, 3), (1024, 512, 32, 1, 4), (1024, 512, 32, 64, 4),
    (1056, 512, 4, 100, 2), (2048, 512, 16, 2, 10), (4096, 1536, 8, 1, 8), (4096, 1536, 3, 49, 2),
    (7168, 2048, 2, 3, 2), (8192, 32, 2, 4, 2), (32, 8192, 2, 4, 2)])
def test_seam(hidden, inter, experts, n, k):
    rng = np.random.default_rng(hidden + inter + n)
    L = Layer(hidden, inter, experts, perm=True)
    x = tokens(rng, n, hidden)
    inds = np.stack([rng.permutation(max(experts, k))[:k] % experts for _ in range(n)]).astype(np.int32)
    y = K.switch_glu(L.g, L.slab.buf, L.table, experts, x, torch.from_numpy(inds).to(DEV))
    ref, b = L.seam(x.double().cpu().numpy(), inds)
    check(y, ref, b)
    again = K.switch_glu(L.g, L.slab.buf, L.table, experts, x, torch.from_numpy(inds).to(DEV))
    assert torch.equal(y, again)


@pytest.mark.parametrize("n", [1, 3, 40, 300])
def test_seam_dropped_absent_and_repeated_ids(n):
    """Ids out of range and experts without a slot give exact zero rows; an id
    twice in a token gives the same row twice; one expert takes every row."""
    rng = np.random.default_rng(n)
    L = Layer(256, 128, 6)
    table = L.table.clone()
    table[4] = -1
    x = tokens(rng, n, 256)
    inds = rng.integers(-2, 8, (n, 4)).astype(np.int32)
    inds[:, 3] = inds[:, 0]
    inds[0] = [-1, 6, 4, -1]
    if n > 2:
        inds[1] = [2, 2, 2, 2]
    y = K.switch_glu(L.g, L.slab.buf, table, 6, x, torch.from_numpy(inds).to(DEV))
    ref, b = L.seam(x.double().cpu().numpy(), np.where(inds == 4, -1, inds))
    check(y, ref, b)
    gone = (inds < 0) | (inds >= 6) | (inds == 4)
    assert (y.cpu()[torch.from_numpy(gone)].view(torch.int16) == 0).all()
    assert torch.equal(y[:, 0], y[:, 3])
    one = torch.full((n, 2), 5, dtype=torch.int32, device=DEV)
    y = K.switch_glu(L.g, L.slab.buf, table, 6, x, one)
    ref, b = L.ffn(5, x.double().cpu().numpy())
    check(y[:, 0], ref, b)
    assert torch.equal(y[:, 0], y[:, 1])


@pytest.mark.parametrize("pin", ["0", "1"])
@pytest.mark.parametrize("hidden,inter,experts,n,k", [
    (128, 128, 2, 1, 1), (128, 256, 3, 50, 2), (256, 128, 3, 200, 2), (640, 384, 2, 129, 1),
    (1024, 512, 4, 140, 2), (384, 640, 2, 300, 2), (4096, 1536, 2, 67, 2), (8192, 128, 1, 20, 1),
    (128, 8192, 1, 20, 1)])
def test_tile_forms(monkeypatch, pin, hidden, inter, experts, n, k):
    """Both forms of the products at both sides of the rule between them: tiles
    of 16 and of 128 rows, with rows that end inside a tile, features that end
    inside a block, dropped ids and an expert without a slot."""
    monkeypatch.setenv("PMOE_MX_TILE", pin)
    rng = np.random.default_rng(hidden + n)
    L = Layer(hidden, inter, experts, perm=True)
    x = tokens(rng, n, hidden)
    inds = rng.integers(0, experts, (n, k)).astype(np.int32)
    inds[rng.random((n, k)) < 0.05] = -1
    table = L.table.clone()
    if experts > 2:
        table[1] = -1
        inds_ref = np.where(inds == 1, -1, inds)
    else:
        inds_ref = inds
    y = K.switch_glu(L.g, L.slab.buf, table, experts, x, torch.from_numpy(inds).to(DEV))
    ref, b = L.seam(x.double().cpu().numpy(), inds_ref)
    check(y, ref, b)
    assert (y.cpu()[torch.from_numpy(inds_ref < 0)].view(torch.int16) == 0).all()
    assert torch.equal(y, K.switch_glu(L.g, L.slab.buf, table, experts, x,
                                       torch.from_numpy(inds).to(DEV)))


@pytest.mark.parametrize("pin", ["0", "1", None])
@pytest.mark.parametrize("hidden,inter,experts,n,k", [
    (32, 32, 3, 40, 2), (96, 224, 2, 300, 1), (160, 544, 3, 150, 2), (544, 160, 2, 130, 2),
    (1440, 288, 3, 70, 2), (288, 1440, 2, 17, 2), (8160, 32, 2, 18, 1), (32, 8160, 2, 18, 1),
    (128, 96, 2, 140, 2), (96, 128, 2, 140, 2)])
def test_tile_forms_of_ragged_reductions(monkeypatch, pin, hidden, inter, experts, n, k):
    """Reductions that end inside a step of 128, from one group to the most, both
    tile heights and what the rule takes: seam and combined outputs, twice the
    same bits, though what the rows' ends lie on differs between the calls."""
    if pin is None:
        monkeypatch.delenv("PMOE_MX_TILE", raising=False)
    else:
        monkeypatch.setenv("PMOE_MX_TILE", pin)
    rng = np.random.default_rng(hidden * 3 + n)
    L = Layer(hidden, inter, experts, perm=True)
    x = tokens(rng, n, hidden)
    inds = rng.integers(0, experts, (n, k)).astype(np.int32)
    w = rng.random((n, k)).astype(np.float32)
    t, wt = torch.from_numpy(inds).to(DEV), torch.from_numpy(w).to(DEV)
    xd = x.double().cpu().numpy()
    y = K.switch_glu(L.g, L.slab.buf, L.table, experts, x, t)
    ref, b = L.seam(xd, inds)
    check(y, ref, b)
    out = K.moe_experts(L.g, L.slab.buf, L.table, experts, x, t, wt)
    ref, b = combined(L, xd, inds, w.astype(np.float64))
    check(out, ref, b)
    # scratch full of bytes that would be NaN as scales
    ws = K.moe_workspace(L.g, n, k, 0, experts, x.device)
    ws.fill_(255)
    _lib.check(_lib.lib().pmoe_moe_workspace_init(ws.data_ptr(), ws.numel(), K._stream()))
    assert torch.equal(y, K.switch_glu(L.g, L.slab.buf, L.table, experts, x, t))
    assert torch.equal(out, K.moe_experts(L.g, L.slab.buf, L.table, experts, x, t, wt))


@pytest.mark.parametrize("hidden,inter,experts,k", [
    (32, 32, 3, 2), (96, 224, 4, 3), (160, 544, 9, 8), (544, 160, 2, 1), (1440, 288, 3, 2),
    (288, 1440, 5, 4), (8160, 32, 2, 1), (32, 8160, 2, 2), (128, 96, 70, 60), (96, 4128, 4, 3)])
def test_one_token_of_ragged_reductions(hidden, inter, experts, k):
    """Both launches of one token where the reductions end inside a step of 128."""
    rng = np.random.default_rng(hidden * 5 + inter)
    L = Layer(hidden, inter, experts, 1, perm=True)
    x = tokens(rng, 1, hidden)
    inds = rng.permutation(experts)[None, :k].astype(np.int32)
    if k > 2:
        inds[0, 1] = -1
    w = rng.random((1, k)).astype(np.float32)
    gate = bf16(rng.standard_normal((1, hidden)) * 0.05)
    t, wt = torch.from_numpy(inds).to(DEV), torch.from_numpy(w).to(DEV)
    xd = x.double().cpu().numpy()
    ref, b = L.seam(xd, inds)
    check(K.switch_glu(L.g, L.slab.buf, L.table, experts, x, t), ref, b)
    out = K.moe_experts(L.g, L.slab.buf, L.table, experts, x, t, wt, L.shared_slot, gate)
    ref, b = combined(L, xd, inds, w.astype(np.float64), gate.double().cpu().numpy())
    check(out, ref, b)


def combined(L, x, inds, w, gate=None):
    y, b = L.seam(x, inds)
    out = (y * w[..., None]).sum(1)
    # each slot's output is rounded to bf16 before the sum
    bo = ((b + np.abs(y) * 2.0 ** -8) * (1 + 2.0 ** -8) * np.abs(w)[..., None]).sum(1)
    if L.shared:
        ys, bs = L.ffn(L.e, x)
        s = 1.0 if gate is None else 1 / (1 + np.exp(-(x @ gate.T)))
        out, bo = out + s * ys, bo + np.abs(s) * (bs + np.abs(ys) * (2.0 ** -8 + 2.0 ** -16))
    return out, bo + 2.0 ** -20 * np.abs(out)


@pytest.mark.parametrize("shared,gated", [(0, False), (1, False), (1, True)])
@pytest.mark.parametrize("hidden,inter,experts,k,n", [
    (96, 64, 4, 2, 1), (1024, 512, 16, 4, 1), (1024, 512, 16, 8, 1), (1024, 512, 16, 8, 2),
    (1024, 512, 16, 4, 21), (544, 160, 8, 3, 130)])
def test_combined(hidden, inter, experts, k, n, shared, gated):
    rng = np.random.default_rng(n + k)
    L = Layer(hidden, inter, experts, shared, perm=True)
    x = tokens(rng, n, hidden)
    inds = np.stack([rng.permutation(experts)[:k] for _ in range(n)]).astype(np.int32)
    if n > 1:
        inds[n // 2, 0] = -1
    w = rng.random((n, k)).astype(np.float32)
    gate = bf16(rng.standard_normal((1, hidden)) * 0.05) if gated else None
    out = K.moe_experts(L.g, L.slab.buf, L.table, experts, x, torch.from_numpy(inds).to(DEV),
                        torch.from_numpy(w).to(DEV), L.shared_slot, gate)
    ref, b = combined(L, x.double().cpu().numpy(), inds, w.astype(np.float64),
                      None if gate is None else gate.double().cpu().numpy())
    check(out, ref, b)


@pytest.mark.parametrize("n", [1, 2, 9, 65, 200])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_blocks_route_as_the_other_format_does(scoring, n):
    """A block's routing does not depend on the experts' format, bit for bit,
    and its output is the combined experts of that routing."""
    rng = np.random.default_rng(n)
    hidden, inter, experts, k = 512, 128, 32, 8
    L = Layer(hidden, inter, experts, 1, perm=False)
    other = SlabStore(_lib.geom(hidden, inter, 4), experts + 1)
    gate_w = bf16(rng.standard_normal((experts, hidden)) * 0.05)
    bias = torch.from_numpy(rng.standard_normal(experts).astype(np.float32) * 0.1).to(DEV)
    x = tokens(rng, n, hidden, big=False)
    rc = K.route_cfg(scoring, experts, k, True, 4, 2, 2.5)
    sb = bias if scoring == "sigmoid" else None
    out, inds, w = K.moe_block(L.g, rc, L.slab.buf, L.table, gate_w, x, score_bias=sb,
                               shared_slot=experts)
    _, inds2, w2 = K.moe_block(other.geom, rc, other.buf, L.table, gate_w, x, score_bias=sb,
                               shared_slot=experts)
    assert torch.equal(inds, inds2) and torch.equal(w, w2)
    ref, b = combined(L, x.double().cpu().numpy(), inds.cpu().numpy(), w.double().cpu().numpy())
    check(out, ref, b)


@pytest.mark.parametrize("n", [1, 4, 100])
def test_bad_rows_stay_their_own(n):
    """An infinity, a NaN or an overflow makes its own row NaN and no other;
    zero rows are exact zeros; tiny and huge rows keep their scale."""
    rng = np.random.default_rng(n)
    L = Layer(256, 128, 2)
    x = torch.cat([tokens(rng, n, 256)] + [tokens(rng, 1, 256) for _ in range(6)])
    base = x.clone()
    x[n, 3], x[n + 1, 200], x[n + 2, 0] = float("inf"), float("nan"), float("-inf")
    x[n + 3] = 0
    x[n + 4] *= 2.0 ** -60
    x[n + 5] *= 2.0 ** 20
    inds = torch.zeros(n + 6, 1, dtype=torch.int32, device=DEV)
    y = K.switch_glu(L.g, L.slab.buf, L.table, 2, x, inds)[:, 0]
    good = K.switch_glu(L.g, L.slab.buf, L.table, 2, base, inds)[:, 0]
    assert torch.isnan(y[n:n + 3]).all()
    assert torch.equal(y[:n], good[:n])
    assert (y[n + 3] == 0).all()
    for r in (n + 4, n + 5):
        ref, b = L.ffn(0, x[r:r + 1].double().cpu().numpy())
        check(y[r:r + 1], ref, b)


def test_bad_scales_reach_their_expert_only():
    """A weight scale of 255 (not a number) makes its expert's rows NaN."""
    rng = np.random.default_rng(0)
    L = Layer(128, 64, 3)
    x = tokens(rng, 6, 128)
    inds = torch.tensor([[0], [1], [2], [0], [1], [2]], dtype=torch.int32, device=DEV)
    good = K.switch_glu(L.g, L.slab.buf, L.table, 3, x, inds)
    L.slab.expert("gate_proj.scales", 1)[5, 2] = 255
    y = K.switch_glu(L.g, L.slab.buf, L.table, 3, x, inds)
    assert torch.isnan(y[[1, 4]]).all() and torch.equal(y[[0, 2, 3, 5]], good[[0, 2, 3, 5]])


@pytest.mark.parametrize("scales", [(1, 3), (60, 63), (180, 184)])
def test_scales_far_from_one(scales):
    rng = np.random.default_rng(0)
    L = Layer(96, 64, 2, scales=scales)
    x = tokens(rng, 5, 96, big=False)
    if scales[0] > 127:
        x = (x.float() * 2.0 ** -40).to(torch.bfloat16)
    if scales[0] < 10:  # products below fp32's range: zeros, never NaN
        inds = torch.zeros(5, 1, dtype=torch.int32, device=DEV)
        assert (K.switch_glu(L.g, L.slab.buf, L.table, 2, x, inds) == 0).all()
        return
    if scales[0] < 127:
        x = (x.float() * 2.0 ** 62).to(torch.bfloat16)
    inds = torch.zeros(5, 1, dtype=torch.int32, device=DEV)
    y = K.switch_glu(L.g, L.slab.buf, L.table, 2, x, inds)[:, 0]
    ref, b = L.ffn(0, x.double().cpu().numpy())
    check(y, ref, b)


def test_rows_do_not_depend_on_the_batch():
    """A row's bits are the same alone among few rows and in another order."""
    rng = np.random.default_rng(3)
    L = Layer(1024, 512, 4)
    x = tokens(rng, 24, 1024)
    inds = torch.from_numpy(rng.integers(0, 4, (24, 2)).astype(np.int32)).to(DEV)
    y = K.switch_glu(L.g, L.slab.buf, L.table, 4, x, inds)
    p = torch.from_numpy(rng.permutation(24)).to(DEV)
    assert torch.equal(K.switch_glu(L.g, L.slab.buf, L.table, 4, x[p], inds[p]), y[p])


def test_custom_slot_layout_and_streams():
    """Components in another order with gaps between them and a longer stride;
    the call on another stream than the default one."""
    rng = np.random.default_rng(5)
    L = Layer(192, 96, 3)
    g = _lib.geom(192, 96, 4, 32)
    order = [7, 6, 3, 4, 0, 1]
    at = 64
    for c in order:
        g.off[c] = at
        at += (g.nbytes[c] + 15) // 16 * 16 + 48
    g.expert_bytes = at + 16
    specs = component_specs(L.g)
    buf = torch.full((3 * g.expert_bytes,), 0xAB, dtype=torch.uint8, device=DEV)
    for e in range(3):
        for c, name in ((0, "gate_proj.weight"), (1, "gate_proj.scales"), (3, "up_proj.weight"),
                        (4, "up_proj.scales"), (6, "down_proj.weight"), (7, "down_proj.scales")):
            nb = specs[name][2]
            dst = e * g.expert_bytes + g.off[c]
            buf[dst:dst + nb] = L.slab.dest(name, e)
    x = tokens(rng, 11, 192)
    inds = torch.from_numpy(rng.integers(0, 3, (11, 2)).astype(np.int32)).to(DEV)
    y = K.switch_glu(L.g, L.slab.buf, L.table, 3, x, inds)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        z = K.switch_glu(g, buf, L.table, 3, x, inds)
    st.synchronize()
    assert torch.equal(y, z)


@pytest.mark.parametrize("hidden,inter,experts,k", [
    (256, 128, 6, 4), (96, 160, 5, 3), (1024, 512, 32, 4), (512, 256, 2, 2)])
@pytest.mark.parametrize("n", [2, 7, 16, 63, 64, 65])
def test_tokens_one_by_one(n, hidden, inter, experts, k):
    """Few tokens of small experts: combined with a gated shared expert, dropped and
    repeated ids and an absent expert; each token's bits are those of its own call."""
    rng = np.random.default_rng(n * hidden)
    L = Layer(hidden, inter, experts, 1, perm=True)
    table = L.table.clone()
    table[0] = -1
    x = tokens(rng, n, hidden)
    inds = rng.integers(-1, experts + 1, (n, k)).astype(np.int32)
    w = rng.random((n, k)).astype(np.float32)
    gate = bf16(rng.standard_normal((1, hidden)) * 0.05)
    t, wt = torch.from_numpy(inds).to(DEV), torch.from_numpy(w).to(DEV)
    seen = np.where(inds == 0, -1, inds)
    xd = x.double().cpu().numpy()
    y = K.switch_glu(L.g, L.slab.buf, table, experts, x, t)
    ref, b = L.seam(xd, seen)
    check(y, ref, b)
    gone = torch.from_numpy((seen < 0) | (seen >= experts))
    assert (y.cpu()[gone].view(torch.int16) == 0).all()
    args = (L.g, L.slab.buf, table, experts)
    out = K.moe_experts(*args, x, t, wt, L.shared_slot, gate)
    ref, b = combined(L, xd, seen, w.astype(np.float64), gate.double().cpu().numpy())
    check(out, ref, b)
    if n <= 7:
        for i in range(n):
            r = slice(i, i + 1)
            assert torch.equal(out[r], K.moe_experts(*args, x[r], t[r], wt[r], L.shared_slot, gate))
            assert torch.equal(y[r], K.switch_glu(*args, x[r], t[r]))


@pytest.mark.parametrize("gap", [1, 2, 4, 8])
@pytest.mark.parametrize("n,pin", [(1, "0"), (20, "0"), (300, "0"), (300, "1")])
def test_scales_anywhere(monkeypatch, n, pin, gap):
    """Scales on no word, on 4 and on 8 bytes give the outputs of scales on 256: the
    forms that fetch them by words and by 16 bytes step aside."""
    monkeypatch.setenv("PMOE_MX_TILE", pin)
    rng = np.random.default_rng(gap)
    hidden, inter = 1024, 512
    L = Layer(hidden, inter, 3)
    g = _lib.geom(hidden, inter, 4, 32)
    specs = component_specs(L.g)
    comps = ((0, "gate_proj.weight"), (1, "gate_proj.scales"), (3, "up_proj.weight"),
             (4, "up_proj.scales"), (6, "down_proj.weight"), (7, "down_proj.scales"))
    at = 0
    for c, name in comps:
        at = (at + 15) // 16 * 16 + (gap if name.endswith("scales") else 0)
        g.off[c] = at
        at += g.nbytes[c]
    g.expert_bytes = (at + 15) // 16 * 16
    buf = torch.full((3 * g.expert_bytes,), 0xFF, dtype=torch.uint8, device=DEV)
    for e in range(3):
        for c, name in comps:
            dst = e * g.expert_bytes + g.off[c]
            buf[dst:dst + specs[name][2]] = L.slab.dest(name, e)
    x = tokens(rng, n, hidden)
    inds = torch.from_numpy(rng.integers(0, 3, (n, 2)).astype(np.int32)).to(DEV)
    want = K.switch_glu(L.g, L.slab.buf, L.table, 3, x, inds)
    assert torch.equal(want, K.switch_glu(g, buf, L.table, 3, x, inds))


def test_slots_past_32_bits():
    """A slot that begins past 4 GiB of the slab gives a near slot's outputs."""
    rng = np.random.default_rng(0)
    L = Layer(1024, 512, 2)
    size = int(L.g.expert_bytes)
    far = (5 << 30) // size
    buf = torch.empty((far + 1) * size, dtype=torch.uint8, device=DEV)
    buf[far * size:] = L.slab.buf[:size]
    buf[(far - 3) * size:(far - 2) * size] = L.slab.buf[size:2 * size]
    table = torch.tensor([far, far - 3], dtype=torch.int32, device=DEV)
    near = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    for n in (1, 5, 400):
        x = tokens(rng, n, 1024)
        inds = torch.from_numpy(np.tile(np.array([[1, 0]], np.int32), (n, 1))).to(DEV)
        assert torch.equal(K.switch_glu(L.g, buf, table, 2, x, inds),
                           K.switch_glu(L.g, L.slab.buf, near, 2, x, inds))


@pytest.mark.parametrize("pin", ["0", "1"])
def test_rows_past_32_bits(monkeypatch, pin):
    """Slot outputs and seam rows of more than 4 GiB: the last rows are those of a
    call of their own."""
    import ctypes
    monkeypatch.setenv("PMOE_MX_TILE", pin)
    hidden, inter, n, k = 8192, 64 if pin == "0" else 128, 36000, 8
    L = Layer(hidden, inter, 3)
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(n, hidden, device=DEV, generator=g).to(torch.bfloat16)
    inds = torch.randint(-1, 3, (n, k), device=DEV, generator=g, dtype=torch.int32)
    w = torch.rand(n, k, device=DEV, generator=g)
    ws = K.moe_workspace(L.g, n, k, 0, 3, x.device, fresh=True)
    out = torch.empty_like(x)
    y = torch.empty(n, k, hidden, device=DEV, dtype=torch.bfloat16)
    lib, p = _lib.lib(), ctypes.byref(L.g)
    args = (p, L.slab.buf.data_ptr(), L.table.data_ptr(), 3, x.data_ptr(), inds.data_ptr())
    _lib.check(lib.pmoe_moe_experts(*args, w.data_ptr(), n, k, -1, None, out.data_ptr(),
                                    ws.data_ptr(), ws.numel(), K._stream()))
    _lib.check(lib.pmoe_switch_glu(*args, n, k, y.data_ptr(), ws.data_ptr(), ws.numel(),
                                   K._stream()))
    for r in (slice(0, 200), slice(n - 200, n)):
        i = inds[r].contiguous()
        assert torch.equal(y[r], K.switch_glu(L.g, L.slab.buf, L.table, 3, x[r].contiguous(), i))
        assert torch.equal(out[r], K.moe_experts(L.g, L.slab.buf, L.table, 3, x[r].contiguous(), i,
                                                 w[r].contiguous()))


@pytest.mark.parametrize("n", [1, 6, 200])
def test_captured_and_replayed(n):
    """A captured call gives the eager bits on every replay, with other work on
    the same workspace between them, and follows its inputs."""
    rng = np.random.default_rng(n)
    L = Layer(512, 256, 8, 1)
    x = tokens(rng, n, 512)
    inds = torch.from_numpy(np.stack([rng.permutation(8)[:4] for _ in range(n)]).astype(np.int32)).to(DEV)
    w = torch.rand(n, 4, device=DEV)

    def go():
        return (K.switch_glu(L.g, L.slab.buf, L.table, 8, x, inds),
                K.moe_experts(L.g, L.slab.buf, L.table, 8, x, inds, w, 8))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, out = go()
    for r in range(4):
        x.copy_(tokens(rng, n, 512))
        inds.copy_(inds.flip(1))
        graph.replay()
        torch.cuda.synchronize()
        y2, out2 = go()
        assert torch.equal(y, y2) and torch.equal(out, out2), r


def test_two_graphs_share_the_workspace():
    """Graphs of different calls and shapes (one token, few rows, several dispatch
    launches, a ragged reduction), replayed in turn with eager calls between."""
    rng = np.random.default_rng(3)
    calls = []
    for hidden, inter, n in ((512, 256, 1), (512, 256, 9), (96, 160, 33), (512, 256, 400)):
        L = Layer(hidden, inter, 6, 1)
        x = tokens(rng, n, hidden)
        inds = torch.from_numpy(rng.integers(-1, 6, (n, 4)).astype(np.int32)).to(DEV)
        w = torch.rand(n, 4, device=DEV)
        calls.append((L, x, lambda L=L, x=x, i=inds, w=w: (
            K.switch_glu(L.g, L.slab.buf, L.table, 6, x, i),
            K.moe_experts(L.g, L.slab.buf, L.table, 6, x, i, w, 6))))
    for _, _, go in reversed(calls):  # the largest workspace first
        go()
    graphs = []
    for _, _, go in calls:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = go()
        graphs.append((graph, outs))
    for r in range(3):
        for _, x, _ in calls:
            x.copy_(tokens(rng, *x.shape))
        for i in rng.permutation(len(calls)):
            graphs[i][0].replay()
            if r == 1:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        for (_, _, go), (_, outs) in zip(calls, graphs):
            assert all(torch.equal(a, b) for a, b in zip(outs, go())), r


def test_two_calls_at_once():
    """Calls on two streams at once, each with a workspace of its own."""
    import ctypes
    rng = np.random.default_rng(4)
    L = Layer(512, 256, 8)
    inds = torch.from_numpy(rng.integers(0, 8, (150, 4)).astype(np.int32)).to(DEV)
    xs = [tokens(rng, 150, 512) for _ in range(2)]
    want = [K.switch_glu(L.g, L.slab.buf, L.table, 8, x, inds) for x in xs]
    ws = [K.moe_workspace(L.g, 150, 4, 0, 8, x.device, fresh=True) for x in xs]
    ys = [torch.empty_like(y) for y in want]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for x, w, y, st in zip(xs, ws, ys, streams):
            _lib.check(_lib.lib().pmoe_switch_glu(
                ctypes.byref(L.g), L.slab.buf.data_ptr(), L.table.data_ptr(), 8, x.data_ptr(),
                inds.data_ptr(), 150, 4, y.data_ptr(), w.data_ptr(), w.numel(), st.cuda_stream))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, ys))


def test_modules_resident_and_paged():
    """QuantizedSwitchGLU(group=32) under a block, resident, then with its
    experts paged through a slab that holds a part of them: the same bits for
    prefill passes and for decode."""
    rng = np.random.default_rng(0)
    hidden, inter, experts, k = 512, 128, 16, 4
    gen = torch.Generator(device=DEV).manual_seed(1)

    def make():
        gen.manual_seed(1)
        glu = S.QuantizedSwitchGLU(hidden, inter, experts, 4, 32, n_shared=1)
        for e in range(experts + 1):
            glu.quantize_expert(e, *(torch.randn(s, device=DEV, generator=gen) * 0.05
                                     for s in ((inter, hidden), (inter, hidden), (hidden, inter))))
        gate = torch.randn(experts, hidden, device=DEV, generator=gen) * 0.1
        sg = torch.randn(1, hidden, device=DEV, generator=gen) * 0.1
        return torch.nn.ModuleList([S.SoftmaxMoEBlock(gate, glu, k, shared_expert_gate=sg)])
    a, b = make(), make()
    cache = S.build_cache_for(b, slots=8)
    S.patch_model(b, cache, predict_mode="off")
    for n in (1, 3, 70):
        x = tokens(rng, n, hidden, big=False)
        ya, yb = a[0](x), b[0](x)
        assert torch.equal(a[0].last_routing[0], b[0].last_routing[0])
        ref = ya.double()
        assert (ya.double() - yb.double()).norm() <= 2.0 ** -7 * ref.norm()
        seam_a = a[0].switch_mlp(x, a[0].last_routing[0])
        seam_b = b[0].switch_mlp(x, a[0].last_routing[0])
        assert torch.equal(seam_a, seam_b)
    assert cache.stats()["evictions"] > 0 or cache.stats()["misses"] > experts


def test_checkpoint_to_output(tmp_path):
    """Experts of a microscaled checkpoint, paged from its bytes, give what the
    64-bit values of those bytes give."""
    from tests.test_mx4 import make_checkpoint
    hidden, inter, experts = 96, 64, 4
    t = make_checkpoint(tmp_path, hidden, inter, experts)
    glu = S.QuantizedSwitchGLU(hidden, inter, experts, 4, 32)
    model = torch.nn.ModuleList([glu])
    cache = S.build_cache_for(model, slots=3, model_path=tmp_path)
    S.patch_model(model, cache, predict_mode="off")
    rng = np.random.default_rng(0)
    x = tokens(rng, 3, hidden)
    inds = torch.tensor([[0, 3], [1, 2], [3, 1]], dtype=torch.int32, device=DEV)
    y = model[0](x, inds).double().cpu().numpy()
    p = "model.layers.0.mlp.switch_mlp."
    for n in range(3):
        for c in range(2):
            e = int(inds[n, c])
            mats = [M.dequant(M.unpack(t[f"{p}{q}.weight"][e]), t[f"{p}{q}.scales"][e])
                    for q in ("gate_proj", "up_proj", "down_proj")]
            ref, b = M.ffn(x[n:n + 1].double().cpu().numpy(), *mats)
            assert (np.abs(y[n, c] - ref[0]) <= b[0] * (1 + 2.0 ** -8) + np.abs(ref[0]) * 2.0 ** -8).all()


@pytest.mark.parametrize("n,k", [(1, 70), (3, 70), (1, 17)])
def test_many_columns(n, k):
    """More columns than a wave has lanes (one token's two launches stop there)."""
    rng = np.random.default_rng(k)
    L = Layer(256, 128, 80, 1)
    x = tokens(rng, n, 256)
    inds = np.stack([rng.permutation(80)[:k] for _ in range(n)]).astype(np.int32)
    inds[0, 3] = -1
    w = rng.random((n, k)).astype(np.float32)
    out = K.moe_experts(L.g, L.slab.buf, L.table, 80, x, torch.from_numpy(inds).to(DEV),
                        torch.from_numpy(w).to(DEV), L.shared_slot, None)
    ref, b = combined(L, x.double().cpu().numpy(), inds, w.astype(np.float64))
    check(out, ref, b)
    y = K.switch_glu(L.g, L.slab.buf, L.table, 80, x, torch.from_numpy(inds).to(DEV))
    ref, b = L.seam(x.double().cpu().numpy(), inds)
    check(y, ref, b)


@pytest.mark.parametrize("n", [1, 5])
def test_overflow_is_nan(n):
    """An intermediate beyond fp32 makes its row NaN, not a plausible number."""
    rng = np.random.default_rng(0)
    L = Layer(256, 128, 2)
    x = tokens(rng, n, 256)
    x[0] = (x[0].float() * 2.0 ** 70).to(torch.bfloat16)
    inds = torch.zeros(n, 1, dtype=torch.int32, device=DEV)
    y = K.switch_glu(L.g, L.slab.buf, L.table, 2, x, inds)
    assert torch.isnan(y[0]).all() and torch.isfinite(y[1:]).all()
    out = K.moe_experts(L.g, L.slab.buf, L.table, 2, x, inds, torch.ones(n, 1, device=DEV))
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1:]).all()


@pytest.mark.parametrize("n", [1, 6])
def test_block_without_allocation(n):
    """pmoe_moe_block_noalloc gives pmoe_moe_block's bits, captured too."""
    import ctypes
    rng = np.random.default_rng(n)
    L = Layer(512, 128, 16, 1)
    x = tokens(rng, n, 512)
    gate_w = bf16(rng.standard_normal((16, 512)) * 0.05)
    rc = K.route_cfg("softmax", 16, 4)
    ref, ri, rw = K.moe_block(L.g, rc, L.slab.buf, L.table, gate_w, x, shared_slot=16)
    out, inds, w = torch.empty_like(ref), torch.empty_like(ri), torch.empty_like(rw)

    def go():
        _lib.check(_lib.lib().pmoe_moe_block_noalloc(
            ctypes.byref(L.g), ctypes.byref(rc), L.slab.buf.data_ptr(), L.table.data_ptr(),
            gate_w.data_ptr(), None, None, x.data_ptr(), n, 16, None, out.data_ptr(),
            inds.data_ptr(), w.data_ptr(), K._stream()))
    go()
    assert torch.equal(out, ref) and torch.equal(inds, ri) and torch.equal(w, rw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for _ in range(3):
        x.copy_(tokens(rng, n, 512))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, K.moe_block(L.g, rc, L.slab.buf, L.table, gate_w, x,
                                            shared_slot=16)[0])


@pytest.mark.parametrize("n", [140, 1500])
def test_large_calls_gate_and_zero_rows(n):
    """Calls whose dispatch takes several launches: the gated shared expert, and the
    seam's zero rows of dropped ids."""
    rng = np.random.default_rng(n)
    L = Layer(256, 128, 6, 1)
    x = tokens(rng, n, 256)
    inds = rng.integers(-1, 7, (n, 8)).astype(np.int32)
    w = rng.random((n, 8)).astype(np.float32)
    gate = bf16(rng.standard_normal((1, 256)) * 0.05)
    t = torch.from_numpy(inds).to(DEV)
    out = K.moe_experts(L.g, L.slab.buf, L.table, 6, x, t, torch.from_numpy(w).to(DEV), 6, gate)
    xd = x.double().cpu().numpy()
    ref, b = combined(L, xd, inds, w.astype(np.float64), gate.double().cpu().numpy())
    check(out, ref, b)
    y = K.switch_glu(L.g, L.slab.buf, L.table, 6, x, t)
    ref, b = L.seam(xd, inds)
    check(y, ref, b)
    gone = torch.from_numpy((inds < 0) | (inds >= 6))
    assert (y.cpu()[gone].view(torch.int16) == 0).all()


def test_calls_whose_arrays_do_not_fit_are_refused():
    L = Layer(256, 128, 4)
    x = tokens(np.random.default_rng(0), 3, 256)
    i, w = torch.zeros(3, 2, dtype=torch.int32, device=DEV), torch.ones(3, 2, device=DEV)
    a = (L.g, L.slab.buf, L.table, 4)
    rc = K.route_cfg("softmax", 4, 2)
    gate_w = torch.zeros(4, 256, device=DEV, dtype=torch.bfloat16)
    for bad in (lambda: K.switch_glu(*a, x[:2], i), lambda: K.switch_glu(*a, x[:, :128].contiguous(), i),
                lambda: K.switch_glu(*a, x.float(), i), lambda: K.switch_glu(*a, x, i.long()),
                lambda: K.switch_glu(*a, x.cpu(), i), lambda: K.switch_glu(*a[:2], L.table[:3], 4, x, i),
                lambda: K.moe_experts(*a, x[:2], i, w), lambda: K.moe_experts(*a, x, i, w[:2]),
                lambda: K.moe_experts(*a, x, i, w[:, :1].contiguous()),
                lambda: K.moe_experts(*a, x, i, w.t()), lambda: K.moe_experts(*a, x, i, w.half()),
                lambda: K.moe_experts(*a, x, i, w, 3, gate_w[:1, :128].contiguous()),
                lambda: K.moe_block(L.g, rc, L.slab.buf, L.table, gate_w[:3], x),
                lambda: K.moe_block(L.g, rc, L.slab.buf, L.table, gate_w, x[:, :128].contiguous()),
                lambda: K.moe_block(L.g, rc, L.slab.buf, L.table[:2], gate_w, x)):
        with pytest.raises((TypeError, ValueError)):
            bad()


def test_empty_call():
    L = Layer(96, 64, 2)
    y = K.switch_glu(L.g, L.slab.buf, L.table, 2, torch.empty(0, 96, dtype=torch.bfloat16, device=DEV),
                     torch.empty(0, 2, dtype=torch.int32, device=DEV))
    assert y.shape == (0, 2, 96)
